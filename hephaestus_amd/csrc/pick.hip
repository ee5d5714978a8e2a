// pick.hip - each row's next token from a batch's logits: penalties for repeated tokens, biases
// and grammar masks, the largest logit and its log-probability, in one pass over the logits.
//
// A workgroup takes a tile of a row. What the rules say about the tile's tokens is gathered in
// LDS first, one word a token, from lists that are short beside the logits: the history, counted
// with integer atomics (the same in any order), and the biases. The logits are in registers
// meanwhile; each is read once, and log-sum-exp's pieces (maximum, sum) of a row's tiles join
// exactly in a second, small launch.
#include <algorithm>

#include "pages.h"

namespace heph {
namespace {

constexpr int kThreads = 512, kVecs = 8, kTile = kThreads * kVecs * 4;

// A token's word: how often it was answered, whether it was seen in the prompt, and the number
// of its bias entry from 1 on.
constexpr uint32_t kCount = 0x7FFFFu, kPrompt = 0x80000u, kSeen = kCount | kPrompt;
constexpr int kBiasShift = 20;
static_assert(HEPH_PICK_MAX_BIAS < 1 << (32 - kBiasShift), "entries have to fit the word");
static_assert(HEPH_ATTN_MAX_KEYS <= (int)kCount, "counts have to fit the word");

struct Part {
    float top, sum;                // the tile's largest l, and sum exp(l - top)
    int at, pad;                   // top's lowest index, -1: none above -inf
};

struct PickArgs {
    int32_t* tokens;
    float* logprob;
    void* out;
    const void* logits;
    Part* parts;
    const int32_t* slots;
    const uint32_t* masks;
    const int32_t* mask_ids;
    int64_t out_stride, logits_stride;
    heph_token_rules rules;
    int rows, vocab, tiles, n_masks, append;
};

typedef int i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4_row __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4_row __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4_row*>(p); }
__device__ __forceinline__ f32x4 load4(const uint16_t* p)
{
    const u16x4_row w = *reinterpret_cast<const u16x4_row*>(p);
    return f32x4{bf16_bits_f32(w[0]), bf16_bits_f32(w[1]), bf16_bits_f32(w[2]), bf16_bits_f32(w[3])};
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const uint16_t* p) { return bf16_bits_f32(*p); }
__device__ __forceinline__ void store4(float* p, const f32x4& x) { *reinterpret_cast<f32x4_row*>(p) = x; }
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& x)
{
    *reinterpret_cast<u16x4_row*>(p) = u16x4_row{f32_to_bf16(x[0]), f32_to_bf16(x[1]), f32_to_bf16(x[2]), f32_to_bf16(x[3])};
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(uint16_t* p, float x) { *p = f32_to_bf16(x); }

__device__ __forceinline__ Part better(const Part& a, const Part& b)
{
    return b.top > a.top || (b.top == a.top && b.at >= 0 && (a.at < 0 || b.at < a.at)) ? b : a;
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// l after its penalties and bias; every operation rounded by itself, as they are stated (a fused
// product and sum would round once).
__device__ __forceinline__ float ruled(float l, uint32_t w, float repetition, float presence, float frequency,
                                       const float* bias)
{
#pragma clang fp contract(off)
    if (w & kSeen) l = l > 0.0f ? l / repetition : l * repetition;
    if (w & kCount) {
        const float lost = (float)(w & kCount) * frequency;
        l = l - (lost + presence);
    }
    if (w >> kBiasShift) l = l + bias[(w >> kBiasShift) - 1];
    return l;
}

template <class T>
__global__ __launch_bounds__(kThreads) void pick_kernel(PickArgs a)
{
    __shared__ __attribute__((aligned(16))) uint32_t words[kTile];
    __shared__ Part best[kThreads / 64];
    __shared__ float sums[kThreads / 64];
    const int tid = threadIdx.x, row = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
    const int base = tile * kTile, n = min(kTile, a.vocab - base);
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride + base;
    f32x4 x[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int i = (k * kThreads + tid) * 4;
        x[k] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 <= n) x[k] = load4(in + i);
        else
            for (int e = 0; e < 3; ++e)
                if (i + e < n) x[k][e] = load1(in + i + e);
    }
    const heph_token_rules& r = a.rules;
    const int slot = a.slots ? a.slots[row] : -1;
    const bool has_rules = a.slots && slot >= 0 && slot < r.n_slots;
    float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
    int n_seen = 0, n_bias = 0, n_prompt = 0;
    if (has_rules) {
        const float* p = r.penalties + (size_t)slot * 3;
        repetition = p[0];
        presence = p[1];
        frequency = p[2];
        if (repetition != 1.0f || presence != 0.0f || frequency != 0.0f) {
            n_seen = min(max(r.length[slot], 0), r.max_tokens);
            n_prompt = r.n_prompt[slot];
        }
        if (r.max_bias > 0) n_bias = min(max(r.n_bias[slot], 0), r.max_bias);
    }
    const float* bias = r.bias + (size_t)(has_rules ? slot : 0) * r.max_bias;
    if (n_seen > 0 || n_bias > 0) {
        for (int i = tid; i < kTile / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int32_t* history = r.history + (size_t)slot * r.max_tokens;
        for (int i = tid; i < n_seen; i += kThreads) {
            const unsigned at = (unsigned)history[i] - (unsigned)base;
            if (at >= (unsigned)n) continue;
            if (i < n_prompt) atomicOr(&words[at], kPrompt);
            else atomicAdd(&words[at], 1u);
        }
        __syncthreads();
        const int32_t* ids = r.bias_ids + (size_t)slot * r.max_bias;
        for (int i = tid; i < n_bias; i += kThreads) {
            const unsigned at = (unsigned)ids[i] - (unsigned)base;
            // (what is below the entry's number stays as it is from here on)
            if (at < (unsigned)n) atomicMax(&words[at], (words[at] & kSeen) | (uint32_t)(i + 1) << kBiasShift);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const uint4 w4 = reinterpret_cast<const uint4*>(words)[k * kThreads + tid];
            if ((w4.x | w4.y | w4.z | w4.w) == 0) continue;
            const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = ruled(x[k][e], ws[e], repetition, presence, frequency, bias);
        }
    }
    const int mask = a.masks && a.mask_ids ? a.mask_ids[row] : -1;
    if (mask >= 0 && mask < a.n_masks) {
        const uint32_t* bits = a.masks + (size_t)mask * ((a.vocab + 31) / 32) + base / 32;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int i = (k * kThreads + tid) * 4;
            if (i >= n) continue;
            const uint32_t b = bits[i / 32] >> (i % 32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(b >> e & 1)) x[k][e] = -INFINITY;
        }
    }
    if (a.out) {
        T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + base;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int i = (k * kThreads + tid) * 4;
            if (i + 4 <= n) store4(out + i, x[k]);
            else
                for (int e = 0; e < 3; ++e)
                    if (i + e < n) store1(out + i + e, x[k][e]);
        }
    }
    Part p{-INFINITY, 0.0f, -1, 0};
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (x[k][e] > p.top) {
                p.top = x[k][e];
                p.at = base + (k * kThreads + tid) * 4 + e;
            }
    for (int m = 32; m; m >>= 1) {
        const Part o{__shfl_xor(p.top, m), 0.0f, __shfl_xor(p.at, m), 0};
        p = better(p, o);
    }
    if ((tid & 63) == 0) best[tid / 64] = p;
    __syncthreads();
    for (int i = 0; i < kThreads / 64; ++i) p = better(p, best[i]);
    const float top = p.top == -INFINITY ? 0.0f : p.top;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += exp_of(x[k][e] - top);
    sum = wave_fold_sum64(sum);
    if ((tid & 63) == 0) sums[tid / 64] = sum;
    __syncthreads();
    if (tid == 0) {
        p.sum = 0.0f;
        for (int i = 0; i < kThreads / 64; ++i) p.sum += sums[i];
        a.parts[blockIdx.x] = p;
    }
}

// One wave a row joins its tiles' parts.
__global__ __launch_bounds__(64) void join_kernel(PickArgs a)
{
    const int row = blockIdx.x, l = threadIdx.x;
    const Part* parts = a.parts + (size_t)row * a.tiles;
    Part p{-INFINITY, 0.0f, -1, 0};
    for (int i = l; i < a.tiles; i += 64) p = better(p, parts[i]);
    for (int m = 32; m; m >>= 1) p = better(p, Part{__shfl_xor(p.top, m), 0.0f, __shfl_xor(p.at, m), 0});
    const float top = p.top == -INFINITY ? 0.0f : p.top;
    float sum = 0.0f;
    for (int i = l; i < a.tiles; i += 64) sum = __builtin_fmaf(parts[i].sum, exp_of(parts[i].top - top), sum);
    sum = wave_fold_sum64(sum);
    if (l != 0) return;
    if (a.tokens) a.tokens[row] = p.at;
    // (no token: the sum is zero, or NaN where there is one)
    if (a.logprob) a.logprob[row] = p.at < 0 && sum == 0.0f ? -INFINITY : -logf(sum);
    if (a.append && p.at >= 0 && a.slots) {
        const int slot = a.slots[row];
        if (slot < 0 || slot >= a.rules.n_slots) return;
        const int n = a.rules.length[slot];
        if (n < 0 || n >= a.rules.max_tokens) return;
        a.rules.history[(size_t)slot * a.rules.max_tokens + n] = p.at;
        a.rules.length[slot] = n + 1;
    }
}

bool sizes_ok(int rows, int vocab) { return rows >= 1 && rows <= (1 << 20) && vocab >= 1 && vocab <= (1 << 24); }
int tiles_of(int vocab) { return (vocab + kTile - 1) / kTile; }

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

size_t heph_pick_ws_bytes(int rows, int vocab)
{
    return sizes_ok(rows, vocab) ? sizeof(Part) * (size_t)rows * tiles_of(vocab) : 0;
}

int heph_pick_tokens(int32_t* tokens, float* logprob, void* out, int64_t out_stride,
                     const void* logits, int64_t logits_stride, int dtype, int rows, int vocab,
                     const heph_token_rules* rules, const int32_t* slots, const uint32_t* masks,
                     int n_masks, const int32_t* mask_ids, int flags, void* ws, size_t ws_bytes,
                     void* stream)
{
    const bool append = flags & HEPH_PICK_APPEND;
    if (!logits || !ws || (!tokens && !out) || (append && (!tokens || !rules || !slots))) return HEPH_ERR_NULL;
    if (rules && slots &&
        (!rules->history || !rules->length || !rules->n_prompt || !rules->penalties ||
         (rules->max_bias > 0 && (!rules->bias_ids || !rules->bias || !rules->n_bias))))
        return HEPH_ERR_NULL;
    if (flags & ~HEPH_PICK_APPEND) return HEPH_ERR_FLAGS;
    if (dtype != HEPH_DTYPE_F32 && dtype != HEPH_DTYPE_BF16) return HEPH_ERR_DTYPE;
    if (!sizes_ok(rows, vocab) || logits_stride < vocab || (out && out_stride < vocab) ||
        (out == logits && out_stride != logits_stride) || (masks && mask_ids && n_masks < 1) ||
        (rules && slots &&
         (rules->n_slots < 1 || rules->max_tokens < 1 || rules->max_tokens > HEPH_ATTN_MAX_KEYS ||
          rules->max_bias < 0 || rules->max_bias > HEPH_PICK_MAX_BIAS)))
        return HEPH_ERR_SHAPE;
    const size_t element = dtype == HEPH_DTYPE_F32 ? 4 : 2;
    if (!aligned(logits, element) || !aligned(out, element) || !aligned(ws, 16)) return HEPH_ERR_ALIGN;
    if (ws_bytes < heph_pick_ws_bytes(rows, vocab)) return HEPH_ERR_WORKSPACE;
    const int64_t blocks = (int64_t)rows * tiles_of(vocab);
    if (blocks > UINT32_MAX / kThreads) return HEPH_ERR_UNSUPPORTED;     // (a launch's most threads)
    if (int st = check_device()) return st;
    PickArgs a{};
    a.tokens = tokens;
    a.logprob = logprob;
    a.out = out;
    a.logits = logits;
    a.parts = static_cast<Part*>(ws);
    a.slots = rules ? slots : nullptr;
    a.masks = masks;
    a.mask_ids = mask_ids;
    a.out_stride = out_stride;
    a.logits_stride = logits_stride;
    if (rules) a.rules = *rules;
    a.rows = rows;
    a.vocab = vocab;
    a.tiles = tiles_of(vocab);
    a.n_masks = n_masks;
    a.append = append;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == HEPH_DTYPE_F32) pick_kernel<float><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else pick_kernel<uint16_t><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    join_kernel<<<rows, 64, 0, s>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
