// pages_scaled.hip - the paged cache with a scale for each block (a page's 64 keys of one kv
// head, K and V apart), found while the block is written; and keys read back from either cache.
//
// The scale is a power of two, 2^e with the least e for which no value is above 448 * 2^e. E4M3
// is a float: its relative precision does not depend on the scale, so a power of two costs
// nothing, makes a change of scale exact (codes times 2^-n, but for those that fall under
// 2^-6, off by at most half of the smallest one's step), and lets the attention's conversions
// multiply by it in passing.
#include "pages_norm.h"

namespace heph {
namespace {

// Exponents for which a code's value, 2^(e-9) to 448 * 2^e, is a normal bf16.
constexpr int kMinExp = -117, kMaxExp = 119;

// Least e with amax <= 448 * 2^e = 1.75 * 2^(e+8): amax's exponent, and one more where its
// mantissa is above 1.75.
__device__ __forceinline__ int exp_of(float amax)
{
    const int e = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 127 - 8;
    return min(max(e, kMinExp), kMaxExp);
}

// The exponent of a scale in memory.
__device__ __forceinline__ int exp_in(float scale)
{
    const int e = (int)((__float_as_uint(scale) >> 23) & 0xFF) - 127;
    return min(max(e, kMinExp), kMaxExp);
}

// x * 2^-e as an E4M3 value; what is no number in E4M3 (NaN, infinities) is NaN.
__device__ __forceinline__ float in_block(float x, int e)
{
    const float y = __builtin_amdgcn_ldexpf(x, -e);
    const float c = fminf(fmaxf(y, -kE4M3Max), kE4M3Max);
    return __builtin_fabsf(x) <= 3.4028234663852886e38f ? c : __uint_as_float(0x7FC00000u);
}

__device__ __forceinline__ uint2 block_codes8(const float* f, int e)
{
    return make_uint2(pack4_e4m3(in_block(f[0], e), in_block(f[1], e), in_block(f[2], e), in_block(f[3], e)),
                      pack4_e4m3(in_block(f[4], e), in_block(f[5], e), in_block(f[6], e), in_block(f[7], e)));
}

// Largest finite |f|.
__device__ __forceinline__ float finite_max8(const float* f, float m)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = __builtin_fabsf(f[i]);
        m = fmaxf(m, a <= 3.4028234663852886e38f ? a : 0.0f);
    }
    return m;
}

// Four codes times f, a power of two.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return pack4_e4m3(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// Bytes e of four dwords.
__device__ __forceinline__ uint32_t column(const uint32_t (&k)[4], int e)
{
    auto byte = [&](uint32_t w) { return w >> (8 * e) & 0xFFu; };
    return byte(k[0]) | byte(k[1]) << 8 | byte(k[2]) << 16 | byte(k[3]) << 24;
}

struct WriteArgs {
    uint16_t* q_out;
    const uint16_t* qkv;
    const uint16_t* q_gamma;
    const uint16_t* k_gamma;
    uint8_t* k_pages;
    uint8_t* v_pages;
    float* scale;
    const float* rope;
    const int32_t* positions;
    const int32_t* slots;
    int64_t q_stride, qkv_stride, n_slots;
    int n_rope, n_tok, n_heads, n_kv;
    float eps;
};

// A wave takes eight query heads of one token.
__device__ __forceinline__ void q_heads(const WriteArgs& a, long unit)
{
    const int blocks = (a.n_heads + 7) / 8, lane = threadIdx.x & 63, c = lane & 7;
    const int t = (int)(unit / blocks), h = (int)(unit % blocks) * 8 + lane / 8;
    if (t >= a.n_tok || h >= a.n_heads) return;        // (whole heads: eight lanes at a time)
    const int pos = a.positions[t];
    const uint16_t* row = a.qkv + t * a.qkv_stride + (size_t)h * kHeadDim + 8 * c;
    const uint4 x_lo = ldg16u(row), x_hi = ldg16u(row + 64);
    const uint4 y_lo = ldg16u(a.q_gamma + 8 * c), y_hi = ldg16u(a.q_gamma + 64 + 8 * c);
    if (pos < 0 || pos >= a.n_rope) return;
    const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * kHeadDim + 16 * c);
    const float4 w[4] = {cs[0], cs[1], cs[2], cs[3]};
    float lo[8], hi[8];
    norm_rope(lo, hi, x_lo, x_hi, y_lo, y_hi, w, a.eps);
    store_head(a.q_out + t * a.q_stride + (size_t)h * kHeadDim + 8 * c, lo, hi);
}

// A workgroup takes the runs of tokens of one page that start among its W tokens, one kv head.
constexpr int kPitch = kHeadDim + 4;               // bytes of a token's codes in LDS
struct WriteLds {
    uint32_t v[kPage * kPitch / 4];
    float amax[2][4];
    int has[kPage];
};

// n <= 64 tokens from t0 on, all of page `page`: lane i's slot and position are token t0 + i's.
__device__ __forceinline__ void write_block(const WriteArgs& a, WriteLds& lds, int h, int t0, int n, int page,
                                            int slot, int pos)
{
    const int tid = threadIdx.x, l = tid & 63, c = tid & 7;
    const size_t at = (size_t)page * a.n_kv + h;
    float* scale = a.scale + (size_t)page * 2 * a.n_kv + h;
    const float old_k = scale[0], old_v = scale[a.n_kv];
    const uint16_t* gamma = a.k_gamma + 8 * c;
    const uint4 y_lo = ldg16u(gamma), y_hi = ldg16u(gamma + 64);
    const int key = slot & (kPage - 1);
    const bool fresh = __ballot(l < n && key == 0) != 0;
    // thread: dims 8c .., 64+8c .. of tokens tid/8 and 32 + tid/8
    float lo[2][8], hi[2][8];
    uint4 v_lo[2], v_hi[2];
    int my_key[2];
    float top_k = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = r * 32 + tid / 8;
        my_key[r] = __shfl(key, i);
        const int p = __shfl(pos, i);
        if (i >= n) continue;
        const uint16_t* row = a.qkv + (int64_t)(t0 + i) * a.qkv_stride + (size_t)(a.n_heads + h) * kHeadDim + 8 * c;
        const uint16_t* v = row + (size_t)a.n_kv * kHeadDim;
        const uint4 x_lo = ldg16u(row), x_hi = ldg16u(row + 64);
        v_lo[r] = ldg16u(v);
        v_hi[r] = ldg16u(v + 64);
        const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)p * kHeadDim + 16 * c);
        const float4 w[4] = {cs[0], cs[1], cs[2], cs[3]};
        norm_rope(lo[r], hi[r], x_lo, x_hi, y_lo, y_hi, w, a.eps);
        top_k = finite_max8(hi[r], finite_max8(lo[r], top_k));
        float f[8];
        unpack8(v_lo[r], f);
        top_v = finite_max8(f, top_v);
        unpack8(v_hi[r], f);
        top_v = finite_max8(f, top_v);
    }
    top_k = wave_fold_max64(top_k);
    top_v = wave_fold_max64(top_v);
    if (l == 0) {
        lds.amax[0][tid / 64] = top_k;
        lds.amax[1][tid / 64] = top_v;
    }
    if (tid < kPage) lds.has[tid] = 0;
    __syncthreads();
    if (tid < n) lds.has[key] = 1;
    auto all = [&](const float (&m)[4]) { return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])); };
    int ek = exp_of(all(lds.amax[0])), ev = exp_of(all(lds.amax[1]));
    uint8_t* kp = a.k_pages + at * kPageBytes;
    uint8_t* vp = a.v_pages + at * kPageBytes;
    if (!fresh) {
        const int was_k = exp_in(old_k), was_v = exp_in(old_v);
        ek = max(ek, was_k);
        ev = max(ev, was_v);
        auto rescale = [&](uint8_t* p, int by) {
            const float f = __builtin_amdgcn_ldexpf(1.0f, by);
            uint4* w = reinterpret_cast<uint4*>(p) + tid;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 x = w[i * 256];
                w[i * 256] = make_uint4(rescale4(x.x, f), rescale4(x.y, f), rescale4(x.z, f), rescale4(x.w, f));
            }
        };
        if (ek > was_k) rescale(kp, was_k - ek);
        if (ev > was_v) rescale(vp, was_v - ev);
    }
    if (tid == 0) {
        scale[0] = __builtin_amdgcn_ldexpf(1.0f, ek);
        scale[a.n_kv] = __builtin_amdgcn_ldexpf(1.0f, ev);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (r * 32 + tid / 8 >= n) continue;
        float f[8];
        uint32_t* to = lds.v + my_key[r] * (kPitch / 4) + 2 * c;
        unpack8(v_lo[r], f);
        uint2 w = block_codes8(f, ev);
        to[0] = w.x;
        to[1] = w.y;
        unpack8(v_hi[r], f);
        w = block_codes8(f, ev);
        to[16] = w.x;
        to[17] = w.y;
    }
    __syncthreads();                               // (the old codes are written too)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (r * 32 + tid / 8 >= n) continue;
        *reinterpret_cast<uint2*>(kp + k_byte(my_key[r], 8 * c)) = block_codes8(lo[r], ek);
        *reinterpret_cast<uint2*>(kp + k_byte(my_key[r], 64 + 8 * c)) = block_codes8(hi[r], ek);
    }
    // V lies key-minor: dims 4g .. 4g+3 of four keys at a time
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(lds.v);
    for (int i = tid; i < 16 * 32; i += 256) {
        const int j = i % 16 * 4, g = i / 16;
        const int has = lds.has[j] | lds.has[j + 1] << 1 | lds.has[j + 2] << 2 | lds.has[j + 3] << 3;
        if (has == 15) {
            uint32_t k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = lds.v[(j + e) * (kPitch / 4) + g];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint32_t*>(vp + v_byte(j, 4 * g + e)) = column(k, e);
        } else if (has) {
            for (int e = 0; e < 4; ++e)
                if (has >> e & 1)
                    for (int d = 4 * g; d < 4 * g + 4; ++d) vp[v_byte(j + e, d)] = bytes[(j + e) * kPitch + d];
        }
    }
    __syncthreads();                               // (LDS is used again)
}

template <int W>
__device__ __forceinline__ void write_window(const WriteArgs& a, long unit)
{
    __shared__ WriteLds lds;
    const int h = (int)(unit % a.n_kv), t0 = (int)(unit / a.n_kv) * W, l = threadIdx.x & 63;
    // lane i: tokens t0 + i and t0 + 64 + i; a token that is not cached has no slot
    auto slot_of = [&](int t, int& pos) {
        if (t < 0 || t >= a.n_tok) return -1;
        const int s = a.slots[t];
        pos = a.positions[t];
        return pos >= 0 && pos < a.n_rope && s >= 0 && s < a.n_slots ? s : -1;
    };
    int pos0 = 0, pos1 = 0, none = 0;
    const int s0 = slot_of(t0 + l, pos0), s1 = slot_of(t0 + 64 + l, pos1);
    const int p0 = s0 >> 6, p1 = s1 >> 6;          // (no slot: -1)
    const int before = slot_of(t0 - 1, none) >> 6, shifted = __shfl_up(p0, 1);
    const int prev = l ? shifted : before;
    for (unsigned long long starts = __ballot(l < W && p0 >= 0 && p0 != prev); starts; starts &= starts - 1) {
        const int s = __ffsll((long long)starts) - 1, page = __builtin_amdgcn_readlane(p0, s);
        const unsigned long long same = __ballot(p0 == page) >> s |
                                        (s ? __ballot(p1 == page) << (64 - s) : 0ull);
        const int n = ~same ? __ffsll((long long)~same) - 1 : 64, i = (l + s) & 63;
        const int a0 = __shfl(s0, i), a1 = __shfl(s1, i), b0 = __shfl(pos0, i), b1 = __shfl(pos1, i);
        write_block(a, lds, h, t0 + s, n, page, l + s < 64 ? a0 : a1, l + s < 64 ? b0 : b1);
    }
}

template <int W>
__global__ __launch_bounds__(256) void write_kernel(WriteArgs a, long page_blocks)
{
    if ((long)blockIdx.x < page_blocks) write_window<W>(a, blockIdx.x);
    else q_heads(a, ((long)blockIdx.x - page_blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// ------------------------------------------------------------------- read ----

struct ReadArgs {
    uint16_t* k_out;
    uint16_t* v_out;
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    const float* kv_scale;         // 2 * n_kv of all pages, or NULL
    const float* page_scale;
    const int32_t* slots;
    int64_t n_slots;
    int n_rows, n_kv;
};

// Eight codes times s as bf16.
__device__ __forceinline__ uint4 bf16_of8(uint2 w, float s)
{
    const uint32_t d[2] = {w.x, w.y};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)d[i], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)d[i], true);
        r[2 * i] = pack2_bf16(lo[0] * s, lo[1] * s);
        r[2 * i + 1] = pack2_bf16(hi[0] * s, hi[1] * s);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// A workgroup takes the runs of consecutive slots of a page that start among its W rows, one kv
// head: V's codes meet in LDS and leave key by key.
template <int W>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a)
{
    __shared__ uint32_t lds[kPage * kPitch / 4];
    const int tid = threadIdx.x, l = tid & 63, h = (int)(blockIdx.x % a.n_kv);
    const int t0 = (int)(blockIdx.x / a.n_kv) * W;
    auto slot_of = [&](int t) {
        if (t < 0 || t >= a.n_rows) return -2;
        const int s = a.slots[t];
        return s >= 0 && s < a.n_slots ? s : -2;
    };
    const int s0 = slot_of(t0 + l), s1 = slot_of(t0 + 64 + l), before = slot_of(t0 - 1);
    const int shifted = __shfl_up(s0, 1), prev = l ? shifted : before;
    for (unsigned long long starts = __ballot(l < W && s0 >= 0 && (s0 != prev + 1 || s0 % kPage == 0)); starts;
         starts &= starts - 1) {
        const int s = __ffsll((long long)starts) - 1, first = __builtin_amdgcn_readlane(s0, s);
        const int page = first / kPage, key0 = first % kPage;
        const unsigned long long in0 = __ballot(s0 >= 0 && s0 - first == l - s), in1 = __ballot(s1 >= 0 && s1 - first == l + 64 - s);
        const unsigned long long same = in0 >> s | (s ? in1 << (64 - s) : 0ull);
        const int n = min(~same ? __ffsll((long long)~same) - 1 : 64, kPage - key0);
        const size_t at = (size_t)page * a.n_kv + h;
        const float* scale = a.kv_scale ? a.kv_scale + h : a.page_scale + (size_t)page * 2 * a.n_kv + h;
        const float sk = scale[0], sv = scale[a.n_kv];
        const uint8_t* kp = a.k_pages + at * kPageBytes;
        const uint8_t* vp = a.v_pages + at * kPageBytes;
        const size_t out = ((size_t)(t0 + s) * a.n_kv + h) * kHeadDim;
        for (int i = tid; i < 16 * 32; i += 256) {
            const int j = i % 16 * 4, g = i / 16;
            if (j + 3 < key0 || j >= key0 + n) continue;
            uint32_t k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = *reinterpret_cast<const uint32_t*>(vp + v_byte(j, 4 * g + e));
#pragma unroll
            for (int e = 0; e < 4; ++e) lds[(j + e) * (kPitch / 4) + g] = column(k, e);
        }
        __syncthreads();
        for (int i = tid; i < n * 16; i += 256) {
            const int r = i / 16, d = i % 16 * 8;
            const size_t o = out + (size_t)r * a.n_kv * kHeadDim + d;
            *reinterpret_cast<uint4*>(a.k_out + o) =
                bf16_of8(*reinterpret_cast<const uint2*>(kp + k_byte(key0 + r, d)), sk);
            const uint32_t* v = lds + (key0 + r) * (kPitch / 4) + d / 4;
            *reinterpret_cast<uint4*>(a.v_out + o) = bf16_of8(make_uint2(v[0], v[1]), sv);
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

int heph_qk_norm_rope_pages_scaled(void* q_out_bf16, int64_t q_stride, const void* qkv_bf16,
                                   int64_t qkv_stride, const void* q_gamma, const void* k_gamma,
                                   uint8_t* k_pages, uint8_t* v_pages, int n_pages, float* page_scale,
                                   const float* rope_table, int n_rope_pos, const int32_t* positions,
                                   const int32_t* slots, int n_tok, int n_heads, int n_kv_heads,
                                   int head_dim, float eps, void* stream)
{
    if (!q_out_bf16 || !qkv_bf16 || !q_gamma || !k_gamma || !k_pages || !v_pages || !page_scale ||
        !rope_table || !positions || !slots)
        return HEPH_ERR_NULL;
    const int64_t heads = (int64_t)n_heads + 2 * (int64_t)n_kv_heads;
    if (!heads_ok(n_heads, n_kv_heads, head_dim) || n_tok < 1 || n_pages < 1 || n_pages >= (1 << 25) ||
        n_rope_pos < 1 || q_stride < (int64_t)n_heads * kHeadDim || qkv_stride < heads * kHeadDim)
        return HEPH_ERR_SHAPE;
    if (!aligned(q_out_bf16, 16) || !aligned(qkv_bf16, 16) || !aligned(q_gamma, 16) ||
        !aligned(k_gamma, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
        !aligned(rope_table, 16) || !aligned(page_scale, 4) || q_stride % 8 || qkv_stride % 8)
        return HEPH_ERR_ALIGN;
    // in place only with the rows where they are: another stride would let one wave overwrite
    // what the next one reads
    if (q_out_bf16 == qkv_bf16 && q_stride != qkv_stride) return HEPH_ERR_SHAPE;
    const int W = n_tok > 512 ? 16 : 1;
    const int64_t page_blocks = ((int64_t)n_tok + W - 1) / W * n_kv_heads;
    const int64_t blocks = page_blocks + ((int64_t)n_tok * ((n_heads + 7) / 8) + 3) / 4;
    if (blocks > UINT32_MAX / 256) return HEPH_ERR_UNSUPPORTED;          // (a launch's most threads)
    if (int st = check_device()) return st;
    WriteArgs a;
    a.q_out = static_cast<uint16_t*>(q_out_bf16);
    a.qkv = static_cast<const uint16_t*>(qkv_bf16);
    a.q_gamma = static_cast<const uint16_t*>(q_gamma);
    a.k_gamma = static_cast<const uint16_t*>(k_gamma);
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.scale = page_scale;
    a.rope = rope_table;
    a.positions = positions;
    a.slots = slots;
    a.q_stride = q_stride;
    a.qkv_stride = qkv_stride;
    a.n_slots = (int64_t)n_pages * kPage;
    a.n_rope = n_rope_pos;
    a.n_tok = n_tok;
    a.n_heads = n_heads;
    a.n_kv = n_kv_heads;
    a.eps = eps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (W == 16) write_kernel<16><<<(unsigned)blocks, 256, 0, s>>>(a, page_blocks);
    else write_kernel<1><<<(unsigned)blocks, 256, 0, s>>>(a, page_blocks);
    return status_of(hipGetLastError());
}

int heph_read_pages(void* k_out_bf16, void* v_out_bf16, const uint8_t* k_pages,
                    const uint8_t* v_pages, int n_pages, const float* kv_scale,
                    const float* page_scale, const int32_t* slots, int n_rows, int n_kv_heads,
                    int head_dim, void* stream)
{
    if (!k_out_bf16 || !v_out_bf16 || !k_pages || !v_pages || !slots || (!kv_scale && !page_scale))
        return HEPH_ERR_NULL;
    if (head_dim != kHeadDim || n_kv_heads < 1 || n_kv_heads > 4096 || n_rows < 1 || n_pages < 1 ||
        n_pages >= (1 << 25) || (kv_scale && page_scale) || k_out_bf16 == v_out_bf16)
        return HEPH_ERR_SHAPE;
    if (!aligned(k_out_bf16, 16) || !aligned(v_out_bf16, 16) || !aligned(k_pages, 16) ||
        !aligned(v_pages, 16))
        return HEPH_ERR_ALIGN;
    const int W = n_rows > 2048 ? 64 : 16;
    const int64_t blocks = ((int64_t)n_rows + W - 1) / W * n_kv_heads;
    if (blocks > UINT32_MAX / 256) return HEPH_ERR_UNSUPPORTED;          // (a launch's most threads)
    if (int st = check_device()) return st;
    ReadArgs a;
    a.k_out = static_cast<uint16_t*>(k_out_bf16);
    a.v_out = static_cast<uint16_t*>(v_out_bf16);
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.kv_scale = kv_scale;
    a.page_scale = page_scale;
    a.slots = slots;
    a.n_slots = (int64_t)n_pages * kPage;
    a.n_rows = n_rows;
    a.n_kv = n_kv_heads;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (W == 64) read_kernel<64><<<(unsigned)blocks, 256, 0, s>>>(a);
    else read_kernel<16><<<(unsigned)blocks, 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
