// pick.hip - each row's next token from a batch's logits: penalties for repeated tokens, biases
// and grammar masks, the largest logit and its log-probability, in one pass over the logits.
//
// A workgroup takes a tile of a row. What the rules say about the tile's tokens is gathered in
// LDS first, one word a token, from lists that are short beside the logits: the history, counted
// with integer atomics (the same in any order), and the biases. The logits are in registers
// meanwhile; each is read once, and log-sum-exp's pieces (maximum, sum) of a row's tiles join
// exactly in a second, small launch.
//
// Measured (vocabulary of 151936 in f32, replayed): bound by memory without rules (256 rows 29.5 us,
// 5.3 TB/s; 64 rows 11.1, with the logits after the rules written 17.0, 4.6 TB/s), by a chain of
// launches and loads for few (three rows 4.8 us, with rules 6.5). Rules add the chain slot, history,
// words: 64 rows with histories of 600 tokens 16.3 us, 256 rows 39.6; histories of 20000, of which
// every tile takes its own tokens, 61, the atomics in LDS. Longer tiles (16384 logits: a row's
// history is read half as often) leave fewer workgroups to hide that chain: 256 rows of 600 tokens
// 48 us, of 20000 75; a workgroup of 1024 threads that loads the next tile ahead 69 and 102.
#include <algorithm>

#include "pages.h"

namespace heph {
namespace {

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
    int rows, vocab, tiles, n_masks, append, by_xcd;
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
// Four logits; PAST: past the caches.
template <bool PAST>
__device__ __forceinline__ void store4(float* p, const f32x4& x)
{
    auto* to = reinterpret_cast<f32x4_row*>(p);
    if constexpr (PAST) __builtin_nontemporal_store(x, to);
    else *to = x;
}
template <bool PAST>
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& x)
{
    const u16x4_row w = {f32_to_bf16(x[0]), f32_to_bf16(x[1]), f32_to_bf16(x[2]), f32_to_bf16(x[3])};
    auto* to = reinterpret_cast<u16x4_row*>(p);
    if constexpr (PAST) __builtin_nontemporal_store(w, to);
    else *to = w;
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(uint16_t* p, float x) { *p = f32_to_bf16(x); }

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// What a sum by `top` counts in one by `all`. (One of nothing is 0, or a NaN that stays one.)
__device__ __forceinline__ float weight(float top, float all) { return top == -INFINITY ? 0.0f : exp_of(top - all); }

// The parts of a wave's lanes as one, in all of them: the largest top, its lowest index, the sums
// by it. (~at orders indexes the other way round, -1 last; equal tops are compared as numbers, so
// that 0 is -0's equal.)
__device__ __forceinline__ Part join_lanes(const Part& p)
{
    Part r;
    r.top = wave_fold_max64(p.top);
    r.at = (int)~lanes_max_u<64>(p.top == r.top ? ~(uint32_t)p.at : 0u);
    r.pad = 0;
    r.sum = wave_fold_sum64(p.sum * weight(p.top, r.top));
    return r;
}

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

// A thread holds V vectors of four logits: a workgroup's tile is 2048 * V of them.
constexpr int kThreads = 512;
constexpr int tile_of(int V) { return kThreads * V * 4; }

// Sixteen tokens of a history in each thread, loaded at once; -1 behind its end.
constexpr int kBatchVecs = 4, kBatch = kBatchVecs * kThreads * 4;
struct Tokens {
    int t[kBatchVecs][4];

    static __device__ __forceinline__ int at(int u) { return (u * kThreads + (int)threadIdx.x) * 4; }
    __device__ __forceinline__ void load(int u, const int32_t* history, int first, int end)
    {
        const int i = first + at(u);
        if (i + 4 <= end) {
            const i32x4_a4 w = *reinterpret_cast<const i32x4_a4*>(history + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[u][e] = w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[u][e] = i + e < end ? history[i + e] : -1;
        }
    }
    // Counted in the words of the tile of n tokens from base on, those from number n_prompt of the
    // history on as answered. A token of another tile goes to a word of its lane's behind the
    // tile's, which costs less than to leave it out (256 rows of 20000 tokens 64 us instead of 74).
    __device__ __forceinline__ void count(uint32_t* words, int spare, int first, int end, int n_prompt, int base,
                                          int n) const
    {
#pragma unroll
        for (int u = 0; u < kBatchVecs; ++u) {
            const int i = first + at(u), low = __builtin_amdgcn_readfirstlane(i);     // the wave's first of 256
            if (low >= end) break;
            uint32_t* word[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned place = (unsigned)t[u][e] - (unsigned)base;
                word[e] = words + (place < (unsigned)n ? place : (unsigned)spare + (threadIdx.x & 63));
            }
            if (low >= n_prompt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) atomicAdd(word[e], 1u);
            } else if (low + 256 <= n_prompt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) atomicOr(word[e], kPrompt);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i + e < n_prompt) atomicOr(word[e], kPrompt);
                    else atomicAdd(word[e], 1u);
                }
            }
        }
    }
};

__device__ __forceinline__ void finish(const PickArgs& a, int row, const Part& p)
{
    if (a.tokens) a.tokens[row] = p.at;
    // (no token: the sum is zero, or NaN where there is one)
    if (a.logprob) a.logprob[row] = p.at < 0 && p.sum == 0.0f ? -INFINITY : -logf(p.sum);
    if (a.append && p.at >= 0 && a.slots) {
        const int slot = a.slots[row];
        if (slot < 0 || slot >= a.rules.n_slots) return;
        const int n = a.rules.length[slot];
        if (n < 0 || n >= a.rules.max_tokens) return;
        a.rules.history[(size_t)slot * a.rules.max_tokens + n] = p.at;
        a.rules.length[slot] = n + 1;
    }
}

template <class T, int V, bool PAST>
__global__ __launch_bounds__(kThreads) void pick_kernel(PickArgs a)
{
    constexpr int kTile = tile_of(V);
    __shared__ __attribute__((aligned(16))) uint32_t words[kTile + 64];
    __shared__ Part waves[kThreads / 64];
    // (workgroups go round the eight XCDs)
    const int tid = threadIdx.x, block = a.by_xcd ? blockIdx.x / 8 : blockIdx.x;
    const int row = a.by_xcd ? block / a.tiles * 8 + (int)(blockIdx.x % 8) : block / a.tiles;
    const int tile = block % a.tiles, base = tile * kTile;
    if (row >= a.rows) return;
    const int n = min(kTile, a.vocab - base);
    // The start is a chain of loads: slot and mask, then what they have, the first tokens of the
    // history (whatever its length) among it; the logits are on their way beside it.
    const int slot = a.slots ? a.slots[row] : -1;
    const int mask_id = a.masks && a.mask_ids ? a.mask_ids[row] : -1;
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride + base;
    float x[V][4];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int i = (k * kThreads + tid) * 4;
        if (i + 4 <= n) {
            const f32x4 w = load4(in + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = i + e < n ? load1(in + i + e) : -INFINITY;
        }
    }
    const bool masked = mask_id >= 0 && mask_id < a.n_masks;
    uint32_t bits[V];
    if (masked) {
        const uint32_t* m = a.masks + (size_t)mask_id * ((a.vocab + 31) / 32) + base / 32;
#pragma unroll
        for (int k = 0; k < V; ++k) bits[k] = m[min((k * kThreads + tid) * 4, n - 1) / 32];
    }
    const heph_token_rules& r = a.rules;
    if (slot >= 0 && slot < r.n_slots) {
        const float* p = r.penalties + (size_t)slot * 3;
        const int32_t* history = r.history + (size_t)slot * r.max_tokens;
        const float repetition = p[0], presence = p[1], frequency = p[2];
        const int n_prompt = r.n_prompt[slot], length = r.length[slot];
        const int n_bias = r.max_bias > 0 ? min(max(r.n_bias[slot], 0), r.max_bias) : 0;
        Tokens batch;
        batch.load(0, history, 0, r.max_tokens);
        const bool neutral = repetition == 1.0f && presence == 0.0f && frequency == 0.0f;
        const int n_seen = neutral ? 0 : min(max(length, 0), r.max_tokens);
        const float* bias = r.bias + (size_t)slot * r.max_bias;
        if (n_seen > 0 || n_bias > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (batch.at(0) + e >= n_seen) batch.t[0][e] = -1;
#pragma unroll
            for (int u = 1; u < kBatchVecs; ++u) batch.load(u, history, 0, n_seen);
            for (int i = tid; i < (n + 3) / 4; i += kThreads)
                reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
            lds_barrier();
            for (int first = 0; first < n_seen; first += kBatch) {
                if (first > 0)
#pragma unroll
                    for (int u = 0; u < kBatchVecs; ++u) batch.load(u, history, first, n_seen);
                batch.count(words, kTile, first, n_seen, n_prompt, base, n);
            }
            lds_barrier();
            if (n_bias > 0) {
                const int32_t* ids = r.bias_ids + (size_t)slot * r.max_bias;
                for (int i = tid; i < n_bias; i += kThreads) {
                    const unsigned at = (unsigned)ids[i] - (unsigned)base;
                    // (what is below the entry's number stays as it is from here on)
                    if (at < (unsigned)n) atomicMax(&words[at], (words[at] & kSeen) | (uint32_t)(i + 1) << kBiasShift);
                }
                lds_barrier();
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int i = (k * kThreads + tid) * 4;
                const uint4 w = reinterpret_cast<const uint4*>(words)[i / 4];
                if (i >= n || (w.x | w.y | w.z | w.w) == 0) continue;
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) x[k][e] = ruled(x[k][e], ws[e], repetition, presence, frequency, bias);
            }
        }
    }
    if (masked) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t b = bits[k] >> (tid * 4 % 32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(b >> e & 1)) x[k][e] = -INFINITY;
        }
    }
    if (a.out) {
        T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + base;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int i = (k * kThreads + tid) * 4;
            if (i + 4 <= n) store4<PAST>(out + i, f32x4{x[k][0], x[k][1], x[k][2], x[k][3]});
            else
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (i + e < n) store1(out + i + e, x[k][e]);
        }
    }
    Part p{-INFINITY, 0.0f, -1, 0};
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (x[k][e] > p.top) {
                p.top = x[k][e];
                p.at = base + (k * kThreads + tid) * 4 + e;
            }
    if (a.logprob) {
        const float by = p.top == -INFINITY ? 0.0f : p.top;
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) p.sum += exp_of(x[k][e] - by);
    }
    p = join_lanes(p);
    if ((tid & 63) == 0) waves[tid / 64] = p;
    lds_barrier();
    if (tid >= 64) return;
    p = join_lanes(tid < kThreads / 64 ? waves[tid] : Part{-INFINITY, 0.0f, -1, 0});
    if (tid != 0) return;
    if (a.tiles == 1) finish(a, row, p);
    else a.parts[(size_t)row * a.tiles + tile] = p;
}

// One wave a row joins its tiles' parts.
__global__ __launch_bounds__(64) void join_kernel(PickArgs a)
{
    const int row = blockIdx.x, l = threadIdx.x;
    const Part* parts = a.parts + (size_t)row * a.tiles;
    Part p{-INFINITY, 0.0f, -1, 0};
    for (int i = l; i < a.tiles; i += 64) {
        // (in order of their indexes: of equal tops the first is kept)
        const Part o = parts[i];
        const float top = fmaxf(p.top, o.top), sum = p.sum * weight(p.top, top) + o.sum * weight(o.top, top);
        if (o.top > p.top) p.at = o.at;
        p.top = top;
        p.sum = sum;
    }
    p = join_lanes(p);
    if (l == 0) finish(a, row, p);
}

bool sizes_ok(int rows, int vocab) { return rows >= 1 && rows <= (1 << 20) && vocab >= 1 && vocab <= (1 << 24); }
int tiles_of(int vocab, int V) { return (vocab + tile_of(V) - 1) / tile_of(V); }

// The longest tile that still gives every CU two workgroups: each of a row's reads its whole history.
// Tiles of 2048, 4096 and 8192, histories of 600 tokens, us: 3 rows 6.4, 6.7, 7.5; 16 rows 10.5, 8.9,
// 9.3; 64 rows 23.2, 17.8, 16.1.
constexpr int kMostVecs = 4, kEnough = 512;
int vecs_of(int rows, int vocab)
{
    int V = kMostVecs;
    while (V > 1 && (int64_t)rows * tiles_of(vocab, V) < kEnough) V /= 2;
    return V;
}

// Parts of as many rows or fewer, of a vocabulary as large or smaller: where a tile is halved, there
// were less than kEnough of the longer ones.
int64_t most_parts(int rows, int vocab)
{
    return std::max<int64_t>((int64_t)rows * tiles_of(vocab, kMostVecs), 2 * kEnough);
}

// With so many rows a row's tiles lie on one XCD, whose L2 then holds its history for all of them
// (histories of 20000 tokens: 64 rows 24.8 -> 23.0 us, 256 rows 64.3 -> 60.9; of 600: the same).
constexpr int kRowsByXcd = 64;
int64_t blocks_of(int rows, int tiles) { return (int64_t)(rows >= kRowsByXcd ? (rows + 7) / 8 * 8 : rows) * tiles; }

// Logits after the rules that the L2s do not hold go past the caches; the others are there for whoever
// reads them next. Ordinary stores and past, us, alone and with a softmax behind them (f32): one row 5.2
// and 5.2, 56 and 68; 16 rows 9.0 and 8.4, 63 and 75; 64 21.2 and 17.0, 102 and 116; 256 63 and 57, 216
// and 184.
constexpr int64_t kL2Bytes = 8 * 4 << 20;

template <class T, bool PAST>
void launch(const PickArgs& a, int V, hipStream_t s)
{
    const unsigned blocks = (unsigned)blocks_of(a.rows, a.tiles);
    if (V == 4) pick_kernel<T, 4, PAST><<<blocks, kThreads, 0, s>>>(a);
    else if (V == 2) pick_kernel<T, 2, PAST><<<blocks, kThreads, 0, s>>>(a);
    else pick_kernel<T, 1, PAST><<<blocks, kThreads, 0, s>>>(a);
    if (a.tiles > 1) join_kernel<<<a.rows, 64, 0, s>>>(a);
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

size_t heph_pick_ws_bytes(int rows, int vocab)
{
    return sizes_ok(rows, vocab) ? sizeof(Part) * (size_t)most_parts(rows, vocab) : 0;
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
    const int V = vecs_of(rows, vocab);
    if (blocks_of(rows, tiles_of(vocab, V)) > UINT32_MAX / kThreads) return HEPH_ERR_UNSUPPORTED;     // (a launch's most threads)
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
    a.tiles = tiles_of(vocab, V);
    a.n_masks = n_masks;
    a.append = append;
    a.by_xcd = rows >= kRowsByXcd;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool past = !out || (int64_t)rows * vocab * (int64_t)element > kL2Bytes;
    if (dtype == HEPH_DTYPE_F32) past ? launch<float, true>(a, V, s) : launch<float, false>(a, V, s);
    else past ? launch<uint16_t, true>(a, V, s) : launch<uint16_t, false>(a, V, s);
    return status_of(hipGetLastError());
}

}  // extern "C"
