// pages_qk.hip - q/k norm per head, rotation and the write of k and v into the
// paged cache for a batch of tokens, and the rotation table it reads.
#include "pages.h"

namespace heph {
namespace {

// Row pos of the table: (cos, sin) of pairs 0..63 in f32, the angle in double
// (an f32 angle at position 2^18 is off by 2^-7). One thread per (pos, pair).
__global__ __launch_bounds__(256) void rope_table_f32_kernel(float2* table, int n_pos, double theta)
{
    constexpr int half = kHeadDim / 2;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)n_pos * half) return;
    const int pos = (int)(i / half), p = (int)(i % half);
    const double angle = (double)pos * pow(theta, -2.0 * (double)p / (double)kHeadDim);
    table[i] = make_float2((float)cos(angle), (float)sin(angle));
}

struct QkArgs {
    uint16_t* q_out;
    const uint16_t* qkv;
    const uint16_t* q_gamma;
    const uint16_t* k_gamma;
    uint8_t* k_pages;
    uint8_t* v_pages;
    const float* kv_inv;
    const float* rope;
    const int32_t* positions;
    const int32_t* slots;
    int64_t q_stride, qkv_stride, n_slots;     // slots fit 31 bits: n_pages < 2^25
    int n_rope, n_tok, n_heads, n_kv;
    float eps;
};

__device__ __forceinline__ void unpack8(const uint4& w, float* f)
{
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16lo(d[i]);
        f[2 * i + 1] = bf16hi(d[i]);
    }
}

__device__ __forceinline__ uint32_t pack2_bf16(float a, float b)
{
    return (uint32_t)f32_to_bf16(a) | (uint32_t)f32_to_bf16(b) << 16;
}

__device__ __forceinline__ float clamp_e4m3(float v) { return fminf(fmaxf(v, -kE4M3Max), kE4M3Max); }

__device__ __forceinline__ uint2 codes8(const float* f, float inv)
{
    return make_uint2(pack4_e4m3(clamp_e4m3(f[0] * inv), clamp_e4m3(f[1] * inv),
                                 clamp_e4m3(f[2] * inv), clamp_e4m3(f[3] * inv)),
                      pack4_e4m3(clamp_e4m3(f[4] * inv), clamp_e4m3(f[5] * inv),
                                 clamp_e4m3(f[6] * inv), clamp_e4m3(f[7] * inv)));
}

// q and k: a wave takes eight heads of one token, eight lanes a head: lane c of them
// holds dims 8c .. 8c+7 and 64+8c .. 64+8c+7, the two halves of eight rotation pairs, in
// two 16-byte loads.
__device__ __forceinline__ void qk_heads(const QkArgs& a, long unit)
{
    const int heads = a.n_heads + a.n_kv, blocks = (heads + 7) / 8;
    const int t = (int)(unit / blocks), lane = threadIdx.x & 63, c = lane & 7;
    const int h = (int)(unit % blocks) * 8 + lane / 8;
    if (t >= a.n_tok || h >= heads) return;            // (whole heads: eight lanes at a time)
    const int pos = a.positions[t];
    const int64_t slot = a.slots[t];
    const bool is_q = h < a.n_heads;
    const uint16_t* row = a.qkv + t * a.qkv_stride + (size_t)h * kHeadDim + 8 * c;
    const uint16_t* gamma = (is_q ? a.q_gamma : a.k_gamma) + 8 * c;
    const uint4 x_lo = ldg16u(row), x_hi = ldg16u(row + 64);
    const uint4 y_lo = ldg16u(gamma), y_hi = ldg16u(gamma + 64);
    if (pos < 0 || pos >= a.n_rope) return;
    const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * kHeadDim + 16 * c);
    const float4 w[4] = {cs[0], cs[1], cs[2], cs[3]};
    float lo[8], hi[8], g_lo[8], g_hi[8];
    unpack8(x_lo, lo);
    unpack8(x_hi, hi);
    unpack8(y_lo, g_lo);
    unpack8(y_hi, g_hi);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(lo[i], lo[i], __builtin_fmaf(hi[i], hi[i], ss));
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor(ss, m);
    const float r = 1.0f / __fsqrt_rn(ss * (1.0f / kHeadDim) + a.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float cc[2] = {w[i].x, w[i].z}, sn[2] = {w[i].y, w[i].w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int e = 2 * i + j;
            const float x = g_lo[e] * (lo[e] * r), y = g_hi[e] * (hi[e] * r);
            lo[e] = x * cc[j] - y * sn[j];
            hi[e] = y * cc[j] + x * sn[j];
        }
    }
    if (is_q) {
        uint16_t* out = a.q_out + t * a.q_stride + (size_t)h * kHeadDim + 8 * c;
        *reinterpret_cast<uint4*>(out) = make_uint4(pack2_bf16(lo[0], lo[1]), pack2_bf16(lo[2], lo[3]),
                                                    pack2_bf16(lo[4], lo[5]), pack2_bf16(lo[6], lo[7]));
        *reinterpret_cast<uint4*>(out + 64) = make_uint4(pack2_bf16(hi[0], hi[1]), pack2_bf16(hi[2], hi[3]),
                                                         pack2_bf16(hi[4], hi[5]), pack2_bf16(hi[6], hi[7]));
    } else if (slot >= 0 && slot < a.n_slots) {
        const int e = h - a.n_heads, key = (int)(slot % kPage);
        const float inv = a.kv_inv[e];
        uint8_t* p = a.k_pages + (size_t)(slot / kPage * a.n_kv + e) * kPageBytes;
        *reinterpret_cast<uint2*>(p + k_byte(key, 8 * c)) = codes8(lo, inv);
        *reinterpret_cast<uint2*>(p + k_byte(key, 64 + 8 * c)) = codes8(hi, inv);
    }
}

// v: a workgroup takes W tokens of one kv head. V lies key-minor, so one token's values
// are single bytes 64 apart; where four tokens fill an aligned run of four slots (a
// prompt's do) their bytes are neighbours. The codes meet in LDS; then sixteen lanes write
// the dwords of up to sixteen such runs, a whole 64-byte line of a dim where the window
// fills a page, and the tokens left over go as bytes. (4096 tokens, 32 + 8 heads, replayed on
// the same rows: in runs 16.4 us, all scattered 45; without any cache write 14.9.)
template <int W>
__device__ __forceinline__ void v_window(const QkArgs& a, long unit)
{
    constexpr int PITCH = kHeadDim + 4;
    __shared__ uint32_t lds[W * PITCH / 4];
    __shared__ int lead_at[16], lead_slot[16], single_at[W], single_slot[W];
    const int h = (int)(unit % a.n_kv), t0 = (int)(unit / a.n_kv) * W, tid = threadIdx.x;
    const int n = min(W, a.n_tok - t0);
    // lane j of each wave: token t0 + j's slot, -1 where there is none to write
    const int l = tid & 63;
    int slot = -1;
    if (l < n) {
        const int pos = a.positions[t0 + l], s = a.slots[t0 + l];
        if (pos >= 0 && pos < a.n_rope && s >= 0 && s < a.n_slots) slot = s;
    }
    const float inv = a.kv_inv[a.n_kv + h];
    const uint16_t* rows = a.qkv + (int64_t)t0 * a.qkv_stride + (size_t)(a.n_heads + a.n_kv + h) * kHeadDim;
    // (all loads at once; past the batch its last row again, not used)
    constexpr int LOADS = (W * 16 + 255) / 256;
    uint4 x[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const int i = min(tid + k * 256, n * 16 - 1);
        x[k] = ldg16u(rows + (int64_t)(i / 16) * a.qkv_stride + i % 16 * 8);
    }
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const int i = tid + k * 256;
        if (i >= n * 16) break;
        float f[8];
        unpack8(x[k], f);
        const uint2 w = codes8(f, inv);
        uint32_t* to = lds + (i / 16) * (PITCH / 4) + i % 16 * 2;
        to[0] = w.x;
        to[1] = w.y;
    }
    bool leads = slot >= 0 && slot % 4 == 0 && l + 3 < W;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const int later = __shfl(slot, min(l + i, 63));       // (by all lanes)
        leads = leads && later == slot + i;
    }
    const unsigned long long lead = __ballot(leads);
    const int first = l - (slot & 3);                  // where slot's run of four would start
    const bool alone = slot >= 0 && !(first >= 0 && (lead >> first & 1));
    const unsigned long long single = __ballot(alone), below = (1ull << l) - 1;
    if (tid < 64) {
        if (leads) {
            lead_at[__popcll(lead & below)] = l;
            lead_slot[__popcll(lead & below)] = slot;
        }
        if (alone) {
            single_at[__popcll(single & below)] = l;
            single_slot[__popcll(single & below)] = slot;
        }
    }
    __syncthreads();
    const int n_lead = __popcll(lead), n_single = __popcll(single), li = tid & 15;
    if (li < n_lead) {
        const int s = lead_slot[li], key = s % kPage;
        uint8_t* p = a.v_pages + ((size_t)(s / kPage) * a.n_kv + h) * kPageBytes;
#pragma unroll
        for (int q = tid / 16; q < kHeadDim / 4; q += 16) {
            uint32_t k[4];                             // dims 4q .. 4q+3 of the run's tokens
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i] = lds[(lead_at[li] + i) * (PITCH / 4) + q];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                auto byte = [&](uint32_t w) { return w >> (8 * e) & 0xFFu; };
                *reinterpret_cast<uint32_t*>(p + v_byte(key, 4 * q + e)) =
                    byte(k[0]) | byte(k[1]) << 8 | byte(k[2]) << 16 | byte(k[3]) << 24;
            }
        }
    }
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(lds);
    for (int i = tid; i < n_single * kHeadDim; i += 256) {
        const int s = single_slot[i / kHeadDim], d = i % kHeadDim;
        uint8_t* p = a.v_pages + ((size_t)(s / kPage) * a.n_kv + h) * kPageBytes;
        p[v_byte(s % kPage, d)] = bytes[single_at[i / kHeadDim] * PITCH + d];
    }
}

// Bound by the stream of qkv and q: 4090 tokens, 32 + 8 heads (94 MB) 19 us, 4.9 TB/s;
// 128 tokens 5.4, 3 tokens 3.8, where a chain of three loads counts. The first v_blocks
// workgroups take v, W tokens each, the others four waves of q and k. A short batch is
// tokens of many sequences, whose bytes are spread over many workgroups. Windows of 4 and
// of 64 tokens, us: 128 scattered tokens 4.1, 7.7, in runs 3.7, 4.1; 512 scattered 7.9, 9.7,
// in runs 5.3, 4.9; 1024 scattered 11.8, 13.6, in runs 8.3, 6.6; 4096 scattered 48, 45, in
// runs 24, 16. Up to 512 tokens the windows of 4 lose no more than 8 %, behind it they lose
// a prompt's runs more and more.
template <int W>
__global__ __launch_bounds__(256) void qk_pages_kernel(QkArgs a, long v_blocks)
{
    if ((long)blockIdx.x < v_blocks) v_window<W>(a, blockIdx.x);
    else qk_heads(a, ((long)blockIdx.x - v_blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

int heph_rope_table_f32(float* table, int n_pos, int head_dim, double theta, void* stream)
{
    if (!table) return HEPH_ERR_NULL;
    if (n_pos < 1 || n_pos > HEPH_ATTN_MAX_KEYS || head_dim != kHeadDim || !(theta > 0.0))
        return HEPH_ERR_SHAPE;
    if (!aligned(table, 16)) return HEPH_ERR_ALIGN;
    if (int st = check_device()) return st;
    const long n = (long)n_pos * (kHeadDim / 2);
    rope_table_f32_kernel<<<(unsigned)((n + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
        reinterpret_cast<float2*>(table), n_pos, theta);
    return status_of(hipGetLastError());
}

int heph_qk_norm_rope_pages(void* q_out_bf16, int64_t q_stride, const void* qkv_bf16,
                            int64_t qkv_stride, const void* q_gamma, const void* k_gamma,
                            uint8_t* k_pages, uint8_t* v_pages, int n_pages,
                            const float* kv_inv_scale, const float* rope_table, int n_rope_pos,
                            const int32_t* positions, const int32_t* slots, int n_tok,
                            int n_heads, int n_kv_heads, int head_dim, float eps, void* stream)
{
    if (!q_out_bf16 || !qkv_bf16 || !q_gamma || !k_gamma || !k_pages || !v_pages ||
        !kv_inv_scale || !rope_table || !positions || !slots)
        return HEPH_ERR_NULL;
    const int64_t heads = (int64_t)n_heads + 2 * (int64_t)n_kv_heads;
    if (!heads_ok(n_heads, n_kv_heads, head_dim) || n_tok < 1 || n_pages < 1 || n_pages >= (1 << 25) || n_rope_pos < 1 ||
        q_stride < (int64_t)n_heads * kHeadDim || qkv_stride < heads * kHeadDim)
        return HEPH_ERR_SHAPE;
    if (!aligned(q_out_bf16, 16) || !aligned(qkv_bf16, 16) || !aligned(q_gamma, 16) ||
        !aligned(k_gamma, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
        !aligned(rope_table, 16) || q_stride % 8 || qkv_stride % 8)
        return HEPH_ERR_ALIGN;
    // in place only with the rows where they are: another stride would let one
    // wave overwrite what the next one reads
    if (q_out_bf16 == qkv_bf16 && q_stride != qkv_stride) return HEPH_ERR_SHAPE;
    const int W = n_tok > 512 ? 64 : 4;
    const int64_t v_blocks = ((int64_t)n_tok + W - 1) / W * n_kv_heads;
    const int64_t blocks = v_blocks + ((int64_t)n_tok * ((n_heads + n_kv_heads + 7) / 8) + 3) / 4;
    if (blocks > INT32_MAX) return HEPH_ERR_UNSUPPORTED;
    if (int st = check_device()) return st;
    QkArgs a;
    a.q_out = static_cast<uint16_t*>(q_out_bf16);
    a.qkv = static_cast<const uint16_t*>(qkv_bf16);
    a.q_gamma = static_cast<const uint16_t*>(q_gamma);
    a.k_gamma = static_cast<const uint16_t*>(k_gamma);
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.kv_inv = kv_inv_scale;
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
    if (W == 64) qk_pages_kernel<64><<<(unsigned)blocks, 256, 0, s>>>(a, v_blocks);
    else qk_pages_kernel<4><<<(unsigned)blocks, 256, 0, s>>>(a, v_blocks);
    return status_of(hipGetLastError());
}

}  // extern "C"
