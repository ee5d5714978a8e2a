// pages_scaled.hip - the paged cache with a scale for each block (a page's 64 keys of one kv
// head, K and V apart), found while the block is written; and keys read back from either cache.
//
// The scale is a power of two, 2^e with the least e for which no value is above 448 * 2^e. E4M3
// is a float: its relative precision does not depend on the scale, so a power of two costs
// nothing, makes a change of scale exact (codes times 2^-n, but for those that fall under
// 2^-6, off by at most half of the smallest one's step), and lets the attention's conversions
// multiply by it in passing.
//
// Measured (32 + 8 heads, graph replays): 4090 tokens of prompts (94 MB with q) 20.8 us, 4.5 TB/s (a
// copy of 1 GiB reaches 5.2), with one scale for all pages 18.9; 128 tokens of as many sequences 6.3
// (4.8), three 4.3 (2.9): there a chain of three loads, the scale's rounds among the lanes and V's
// single bytes count. 65001 rows read back (399 MB) in 79 us, 5.0 TB/s.
#include <algorithm>

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

// Codes of eight values times f = 2^-e; what is no number in E4M3 (NaN, infinities) is NaN.
__device__ __forceinline__ float in_block(float x, float f)
{
    const float y = __builtin_amdgcn_fmed3f(x * f, -kE4M3Max, kE4M3Max);
    return __builtin_fabsf(x) <= 3.4028234663852886e38f ? y : __uint_as_float(0x7FC00000u);
}

__device__ __forceinline__ uint2 block_codes8(const float* x, float f)
{
    return make_uint2(pack4_e4m3(in_block(x[0], f), in_block(x[1], f), in_block(x[2], f), in_block(x[3], f)),
                      pack4_e4m3(in_block(x[4], f), in_block(x[5], f), in_block(x[6], f), in_block(x[7], f)));
}

// 2^-e of a block's e: a normal float.
__device__ __forceinline__ float inverse(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }

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

// A wave takes 8 * B query heads of one token: their loads are all on their way at once, which
// keeps memory busy with the few waves that the blocks' registers leave (4090 tokens, 32 heads, with
// ordinary stores: B = 1 27.0 us, 2 24.7, 4 24.3). A long batch's q (B > 1) goes past the caches: 20.5 us
// (B = 4 21.0; 2048 scattered tokens 78 and 84). With the attention behind the write both take
// the same (8 prompts of 512 tokens 75.0 us, 74.4 with ordinary stores; 16 of 1024 296, 297).
template <int B>
__device__ __forceinline__ void q_heads(const WriteArgs& a, long unit)
{
    const int groups = (a.n_heads + 8 * B - 1) / (8 * B), lane = threadIdx.x & 63, c = lane & 7;
    const int t = (int)(unit / groups), first = (int)(unit % groups) * 8 * B + lane / 8;
    if (t >= a.n_tok) return;
    const int pos = a.positions[t];
    const uint16_t* row = a.qkv + t * a.qkv_stride + 8 * c;
    uint4 x_lo[B], x_hi[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const uint16_t* p = row + (size_t)min(first + 8 * i, a.n_heads - 1) * kHeadDim;
        x_lo[i] = ldg16u(p);
        x_hi[i] = ldg16u(p + 64);
    }
    const uint4 y_lo = ldg16u(a.q_gamma + 8 * c), y_hi = ldg16u(a.q_gamma + 64 + 8 * c);
    if (pos < 0 || pos >= a.n_rope) return;
    const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * kHeadDim + 16 * c);
    const float4 w[4] = {cs[0], cs[1], cs[2], cs[3]};
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const int h = first + 8 * i;
        if (h >= a.n_heads) return;                // (whole heads: eight lanes at a time)
        float lo[8], hi[8];
        norm_rope(lo, hi, x_lo[i], x_hi[i], y_lo, y_hi, w, a.eps);
        store_head<(B > 1)>(a.q_out + t * a.q_stride + (size_t)h * kHeadDim + 8 * c, lo, hi);
    }
}

// One thread's part of a token: sixteen values of k (normalized and rotated), dims 8c .. and
// 64+8c .., or of v. K and V of a block have nothing to do with each other: different workgroups
// take them (a wave for both: 128 tokens 7.0 us instead of 6.1, three 5.4 instead of 4.1).
template <bool V>
struct Values {
    float lo[8], hi[8];
    uint4 w_lo, w_hi;              // v as it came

    // Token t's, and the largest finite magnitude.
    __device__ __forceinline__ float load(const WriteArgs& a, int h, int64_t t, int pos, int c)
    {
        const uint16_t* p = a.qkv + t * a.qkv_stride + (size_t)(a.n_heads + (V ? a.n_kv : 0) + h) * kHeadDim + 8 * c;
        w_lo = ldg16u(p);
        w_hi = ldg16u(p + 64);
        if constexpr (V) {
            unpack8(w_lo, lo);
            unpack8(w_hi, hi);
        } else {
            const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * kHeadDim + 16 * c);
            const float4 w[4] = {cs[0], cs[1], cs[2], cs[3]};
            const uint4 y_lo = ldg16u(a.k_gamma + 8 * c), y_hi = ldg16u(a.k_gamma + 64 + 8 * c);
            norm_rope(lo, hi, w_lo, w_hi, y_lo, y_hi, w, a.eps);
        }
        return finite_max8(hi, finite_max8(lo, 0.0f));
    }
    // Codes of the two eights under 2^e.
    __device__ __forceinline__ void codes(uint2 (&w)[2], int e)
    {
        if constexpr (V) {         // (unpacked again: fewer registers while the block's scale is found)
            unpack8(w_lo, lo);
            unpack8(w_hi, hi);
        }
        w[0] = block_codes8(lo, inverse(e));
        w[1] = block_codes8(hi, inverse(e));
    }
};

// A block: its codes, its scale, and the exponent that the scale had.
template <bool V>
struct Block {
    uint8_t* codes;
    float* scale;
    int was;

    __device__ __forceinline__ Block(const WriteArgs& a, int page, int h)
        : codes((V ? a.v_pages : a.k_pages) + ((size_t)page * a.n_kv + h) * kPageBytes),
          scale(a.scale + (size_t)page * 2 * a.n_kv + (V ? a.n_kv : 0) + h), was(exp_in(*scale))
    {
    }
    // Its exponent with new values up to top.
    __device__ __forceinline__ int grow(float top, bool fresh) const
    {
        const int e = exp_of(top);
        return fresh ? e : max(e, was);
    }
    // The codes that are there divided by 2^(e - was), by THREADS threads.
    template <int THREADS>
    __device__ __forceinline__ void rescale(int e, int tid) const
    {
        const float f = __builtin_amdgcn_ldexpf(1.0f, was - e);
        uint4* w = reinterpret_cast<uint4*>(codes) + tid;
#pragma unroll 1
        for (int i = 0; i < kPageBytes / 16; i += THREADS) {
            const uint4 x = w[i];
            w[i] = make_uint4(rescale4(x.x, f), rescale4(x.y, f), rescale4(x.z, f), rescale4(x.w, f));
        }
    }
    __device__ __forceinline__ void store_scale(int e) const { *scale = __builtin_amdgcn_ldexpf(1.0f, e); }
    __device__ __forceinline__ void store_k(int key, int c, const uint2 (&w)[2]) const
    {
        *reinterpret_cast<uint2*>(codes + k_byte(key, 8 * c)) = w[0];
        *reinterpret_cast<uint2*>(codes + k_byte(key, 64 + 8 * c)) = w[1];
    }
};

constexpr int kPitch = kHeadDim + 4;               // bytes of a token's codes in LDS
struct WriteLds {
    uint32_t v[kPage * kPitch / 4];
    float top[8];
    int has[kPage];
};

// n <= 8 tokens from t0 on, all of page `page`, by one wave: slot and pos are those of this lane's
// token, t0 + l/8; fresh: key 0 is among them. V's codes leave as single bytes.
template <bool V>
__device__ __forceinline__ void write_few(const WriteArgs& a, int h, int t0, int n, int page, bool fresh, int slot,
                                          int pos)
{
    const int l = threadIdx.x & 63, c = l & 7, i = l / 8, key = slot & (kPage - 1);
    const Block<V> block(a, page, h);
    Values<V> x;
    float top = 0.0f;
    if (i < n) top = x.load(a, h, t0 + i, pos, c);
    const int e = block.grow(wave_fold_max64(top), fresh);
    if (!fresh && e > block.was) {
        block.template rescale<64>(e, l);
        wait_vm<0>();                              // (the new codes come behind)
    }
    if (l == 0) block.store_scale(e);
    if (i >= n) return;
    uint2 w[2];
    x.codes(w, e);
    if constexpr (V) {
        uint8_t* to = block.codes + v_byte(key, 8 * c);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int d = 0; d < 8; ++d)
                to[half * 4096 + d * 64] = (uint8_t)((d < 4 ? w[half].x : w[half].y) >> (d % 4 * 8));
    } else {
        block.store_k(key, c, w);
    }
}

// The same for n <= 64 by the workgroup: token i is row row_of(i), lane i has its slot and position.
template <int THREADS, bool V, class Row>
__device__ __forceinline__ void write_block(const WriteArgs& a, WriteLds& lds, int h, Row row_of, int n, int page,
                                            bool fresh, int slot, int pos)
{
    constexpr int R = 512 / THREADS;               // a thread's tokens: tid/8, and every THREADS/8-th
    const int tid = threadIdx.x, l = tid & 63, c = tid & 7, key = slot & (kPage - 1);
    const Block<V> block(a, page, h);
    Values<V> x[R];
    int my_key[R];
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = r * (THREADS / 8) + tid / 8;
        my_key[r] = __shfl(key, i);
        const int p = __shfl(pos, i), t = row_of(i);
        if (i < n) top = fmaxf(top, x[r].load(a, h, t, p, c));
    }
    top = wave_fold_max64(top);
    if (tid < kPage) lds.has[tid] = 0;
    if (l == 0) lds.top[tid / 64] = top;
    __syncthreads();
    if (tid < n) lds.has[key] = 1;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) top = fmaxf(top, lds.top[i]);
    const int e = block.grow(top, fresh);
    if (!fresh && e > block.was) {                 // (the same in all threads)
        block.template rescale<THREADS>(e, tid);
        __syncthreads();                           // (the new codes come behind)
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r * (THREADS / 8) + tid / 8 >= n) continue;
        uint2 w[2];
        x[r].codes(w, e);
        if constexpr (V) {
            uint32_t* to = lds.v + my_key[r] * (kPitch / 4) + 2 * c;
            to[0] = w[0].x;
            to[1] = w[0].y;
            to[16] = w[1].x;
            to[17] = w[1].y;
        } else {
            block.store_k(my_key[r], c, w);
        }
    }
    __syncthreads();                               // (the scale is read by all)
    if (tid == 0) block.store_scale(e);
    if constexpr (V) {
        // V lies key-minor: dims 4g .. 4g+3 of four keys at a time
        const uint8_t* bytes = reinterpret_cast<const uint8_t*>(lds.v);
#pragma unroll
        for (int i = tid; i < 16 * 32; i += THREADS) {
            const int j = i % 16 * 4, g = i / 16;
            const int has = lds.has[j] | lds.has[j + 1] << 1 | lds.has[j + 2] << 2 | lds.has[j + 3] << 3;
            if (has == 15) {
                uint32_t k[4];
#pragma unroll
                for (int d = 0; d < 4; ++d) k[d] = lds.v[(j + d) * (kPitch / 4) + g];
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<uint32_t*>(block.codes + v_byte(j, 4 * g + d)) = column(k, d);
            } else if (has) {
#pragma unroll 1
                for (int k = 0; k < 4; ++k)
                    if (has >> k & 1)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
                            block.codes[v_byte(j + k, 4 * g + d)] = bytes[(j + k) * kPitch + 4 * g + d];
            }
        }
        __syncthreads();                           // (LDS is used again)
    }
}

// Token t's slot; -1: it is not cached, or not there.
__device__ __forceinline__ int slot_of(const WriteArgs& a, int64_t t, int& pos)
{
    const int64_t at = min(max(t, (int64_t)0), (int64_t)a.n_tok - 1);
    const int s = a.slots[at];
    pos = a.positions[at];
    return (t >= 0) & (t < a.n_tok) & (pos >= 0) & (pos < a.n_rope) & (s >= 0) & (s < a.n_slots) ? s : -1;
}

// The page of the nearest cached token from token t on, upwards (step 1) or downwards (-1); -1: none.
// (512 tokens' loads at once: the padding behind a batch may be long.)
__device__ __forceinline__ int page_near(const WriteArgs& a, int64_t t, int step)
{
    constexpr int K = 8;
    for (; t >= 0 && t < a.n_tok; t += 64 * K * step) {
        int slot[K], pos;
#pragma unroll
        for (int k = 0; k < K; ++k) slot[k] = slot_of(a, t + step * (64 * k + (int)(threadIdx.x & 63)), pos);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const unsigned long long there = __ballot(slot[k] >= 0);
            if (there) return __builtin_amdgcn_readlane(slot[k] >> 6, __ffsll((long long)there) - 1);
        }
    }
    return -1;
}

// The tokens of a page from token t on with others among them that are not cached: how many, and
// lane i's row, slot and position of the i-th.
__device__ __forceinline__ int sparse_run(const WriteArgs& a, int t, int page, int& row, int& slot, int& pos)
{
    const int l = threadIdx.x & 63;
    int n = 0;
    for (int64_t first = t; first < a.n_tok && n < kPage; first += 64) {
        int p;
        const int s = slot_of(a, first + l, p);
        const unsigned long long other = __ballot(s >= 0 && s >> 6 != page);
        const unsigned long long mine = __ballot(s >= 0 && s >> 6 == page) & (other ? (other & -other) - 1 : ~0ull);
        // lane n + k takes what the k-th of these lanes has
        unsigned long long m = mine;
#pragma unroll 1
        for (int k = n; k < l; ++k) m &= m - 1;
        const int from = m ? __ffsll((long long)m) - 1 : 0, from_slot = __shfl(s, from), from_pos = __shfl(p, from);
        if (l >= n && m) {
            row = (int)first + from;
            slot = from_slot;
            pos = from_pos;
        }
        n = min(n + __popcll(mine), kPage);
        if (other) break;
    }
    return n;
}

// A workgroup takes K or V of one kv head of the runs of tokens of one page that start among its W
// tokens: each run of up to eight by a wave, then the longer ones by all of them. No other one
// touches those blocks, so that a scale and the codes under it change without an atomic. Tokens that
// are not cached neither end a run nor belong to one: a window with such among a run's is written
// run by run (512 tokens of a prompt 8.9 us, with every eighth skipped 13.6). To look for them costs
// batches without any nothing or little (4090 tokens 20.8 us instead of 20.2).
template <int THREADS, int W, bool V>
__device__ __forceinline__ void write_window(const WriteArgs& a, WriteLds& lds, int h, int t0)
{
    const int l = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // lane i: tokens t0 + i and t0 + 64 + i (all loads at once); a token that is not cached has no slot
    const int u0 = t0 + l, u1 = u0 + 64, ub = t0 - 1, last = a.n_tok - 1;
    int s0 = a.slots[min(u0, last)], s1 = a.slots[min(u1, last)], sb = a.slots[max(ub, 0)];
    const int pos0 = a.positions[min(u0, last)], pos1 = a.positions[min(u1, last)], posb = a.positions[max(ub, 0)];
    auto cached = [&](int t, int s, int pos) {
        return (t >= 0) & (t <= last) & (pos >= 0) & (pos < a.n_rope) & (s >= 0) & (s < a.n_slots);
    };
    s0 = cached(u0, s0, pos0) ? s0 : -1;
    s1 = cached(u1, s1, pos1) ? s1 : -1;
    sb = cached(ub, sb, posb) ? sb : -1;
    const int p0 = s0 >> 6, p1 = s1 >> 6;          // (no slot: -1)
    if (__builtin_expect(__any((p0 < 0 && u0 <= last) || (p1 < 0 && u1 <= last) || (sb < 0 && t0 > 0)), 0)) {
        const unsigned long long there0 = __ballot(p0 >= 0), there1 = __ballot(p1 >= 0);
        if (!(there0 << (64 - W))) return;         // (none starts here)
        const int before = sb >= 0 ? sb >> 6 : page_near(a, (int64_t)t0 - 2, -1);
        const unsigned long long below0 = there0 & ((1ull << l) - 1), below1 = there1 & ((1ull << l) - 1);
        // the page of the last cached token before the lane's two
        const int in0 = __shfl(p0, 63 - __clzll((long long)(below0 | 1))), end0 = __shfl(p0, 63 - __clzll((long long)(there0 | 1)));
        const int in1 = __shfl(p1, 63 - __clzll((long long)(below1 | 1)));
        const int prev0 = below0 ? in0 : before, prev1 = below1 ? in1 : there0 ? end0 : before;
        // behind these 128 tokens, is there more of a run that starts here?
        const int end = there1 ? __shfl(p1, 63 - __clzll((long long)there1)) : end0;
        const bool open = !(there1 >> 63) && __any(l < W && p0 == end) && page_near(a, (int64_t)t0 + 128, 1) == end;
        const bool gap0 = p0 >= 0 && p0 == prev0 && (l ? !(there0 >> (l - 1) & 1) : sb < 0);
        const bool gap1 = p1 >= 0 && p1 == prev1 && (l ? !(there1 >> (l - 1) & 1) : !(there0 >> 63));
        if (__any(gap0 | gap1 | open)) {
            for (unsigned long long starts = __ballot(l < W && p0 >= 0 && p0 != prev0); starts; starts &= starts - 1) {
                const int s = __ffsll((long long)starts) - 1, page = __builtin_amdgcn_readlane(p0, s);
                int row = 0, slot = 0, pos = 0;
                const int n = sparse_run(a, t0 + s, page, row, slot, pos);
                const bool begins = __any(l < n && (slot & (kPage - 1)) == 0);
                write_block<THREADS, V>(a, lds, h, [&](int i) { return __shfl(row, i); }, n, page, begins, slot, pos);
            }
            return;
        }
    }
    const int shifted = __builtin_amdgcn_update_dpp(sb >> 6, p0, 0x138, 0xF, 0xF, false);     // the lane below's
    unsigned long long starts = __ballot(l < W && p0 >= 0 && p0 != shifted), more = 0;
    // The run that starts at lane s: its page and tokens, and lane i's slot and position of its i-th.
    auto page_of = [&](int s) { return __builtin_amdgcn_readlane(p0, s); };
    auto from = [](int s, unsigned long long m0, unsigned long long m1) { return m0 >> s | (s ? m1 << (64 - s) : 0ull); };
    auto length = [&](int s) {
        const int page = page_of(s);
        const unsigned long long same = from(s, __ballot(p0 == page), __ballot(p1 == page));
        return ~same ? __ffsll((long long)~same) - 1 : 64;
    };
    const unsigned long long first0 = __ballot((s0 & (kPage - 1)) == 0), first1 = __ballot((s1 & (kPage - 1)) == 0);
    auto fresh = [&](int s, int n) { return (from(s, first0, first1) << (64 - n)) != 0; };
    // token i of the run's value
    auto of_run = [&](int s, int i, int v0, int v1) {
        const int a0 = __shfl(v0, (i + s) & 63);
        const int a1 = __shfl(v1, (i + s) & 63);
        return i + s < 64 ? a0 : a1;
    };
    for (int k = 0; starts; starts &= starts - 1) {
        const int s = __ffsll((long long)starts) - 1, n = length(s);
        if (n > 8) more |= 1ull << s;
        else if (k++ % (THREADS / 64) == wave)
            write_few<V>(a, h, t0 + s, n, page_of(s), fresh(s, n), of_run(s, l / 8, s0, s1), of_run(s, l / 8, pos0, pos1));
    }
    for (; more; more &= more - 1) {
        const int s = __ffsll((long long)more) - 1, n = length(s);
        write_block<THREADS, V>(a, lds, h, [&](int i) { return t0 + s + i; }, n, page_of(s), fresh(s, n), of_run(s, l, s0, s1), of_run(s, l, pos0, pos1));
    }
}

// Every q_every-th workgroup takes query heads, the others windows of tokens, until either are done:
// the blocks wait for their loads while q streams (4090 tokens, all windows first 43 us, all q
// first 41, in turn 31, each with windows of 16 and 32 heads a wave). Three workgroups of 512 threads
// a CU: they leave 80 registers, with two the same 4090 tokens take 22.4 us instead of 20.2.
template <int THREADS, int W, int B>
__global__ __launch_bounds__(THREADS, THREADS == 512 ? 6 : 4) void write_kernel(WriteArgs a, int q_every, int page_blocks)
{
    const int b = blockIdx.x, turn = b / q_every;
    const bool is_q = b % q_every == 0;
    if (!is_q) {
        __shared__ WriteLds lds;
        const int unit = b - turn - 1, index = unit % (2 * a.n_kv), t0 = unit / (2 * a.n_kv) * W;
        if (unit >= page_blocks) return;
        if (index < a.n_kv) write_window<THREADS, W, false>(a, lds, index, t0);
        else write_window<THREADS, W, true>(a, lds, index - a.n_kv, t0);
    } else {
        q_heads<B>(a, (long)turn * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    }
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
// head: V's codes meet in LDS and leave key by key. Bound by the rows' 16-bit stores, which go past
// the caches (65001 rows 79 us instead of 85, and 146 instead of 151 with an addition of k and v behind
// them; 100 and 1000 rows the same, alone and with it).
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
        // (all of the block's loads at once; past the run its last piece again, not used)
        uint2 k_codes[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(tid + u * 256, n * 16 - 1);
            k_codes[u] = *reinterpret_cast<const uint2*>(kp + k_byte(key0 + i / 16, i % 16 * 8));
        }
#pragma unroll
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
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = tid + u * 256, r = i / 16, d = i % 16 * 8;
            if (r >= n) break;
            const size_t o = out + (size_t)r * a.n_kv * kHeadDim + d;
            store_past(a.k_out + o, bf16_of8(k_codes[u], sk));
            const uint32_t* v = lds + (key0 + r) * (kPitch / 4) + d / 4;
            store_past(a.v_out + o, bf16_of8(make_uint2(v[0], v[1]), sv));
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
    // A long batch takes windows of 64 tokens, a prompt's page to a workgroup of 512 threads; a
    // shorter one windows of 4, more workgroups. Windows of 4 and of 64, us: 512 tokens of as many
    // sequences 13.7, 23.6, in runs 8.8, 7.2; 1024 scattered 28, 38, in runs 12.9, 10.4; 2048 scattered
    // 76, 80, in runs 20.6, 12.7; 4090 in runs 39, 19.0.
    const bool many = n_tok > 1024;
    const int W = many ? 64 : 4, waves = many ? 8 : 4, heads_a_wave = many ? 16 : 8;
    const int64_t page_blocks = ((int64_t)n_tok + W - 1) / W * 2 * n_kv_heads;
    const int64_t q_blocks = ((int64_t)n_tok * ((n_heads + heads_a_wave - 1) / heads_a_wave) + waves - 1) / waves;
    // one q block and then q_every - 1 of pages, in turn
    const int64_t pages_a_turn = std::max<int64_t>((page_blocks + q_blocks / 2) / q_blocks, 1), q_every = 1 + pages_a_turn;
    const int64_t turns = std::max(q_blocks, (page_blocks + pages_a_turn - 1) / pages_a_turn), blocks = turns * q_every;
    if (blocks > UINT32_MAX / 512) return HEPH_ERR_UNSUPPORTED;          // (a launch's most threads)
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
    if (many) write_kernel<512, 64, 2><<<(unsigned)blocks, 512, 0, s>>>(a, (int)q_every, (int)page_blocks);
    else write_kernel<256, 4, 1><<<(unsigned)blocks, 256, 0, s>>>(a, (int)q_every, (int)page_blocks);
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
    // Windows of 16 rows and of 64, us: 100 rows 4.0, 5.3; 1000 5.4, 6.1; 2000 5.8, 5.7, scattered 26,
    // 59; 4000 8.8, 8.0; 65001 168, 77.
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
