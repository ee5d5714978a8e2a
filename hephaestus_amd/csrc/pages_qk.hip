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
    int64_t q_stride, qkv_stride, n_slots;
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

// A wave takes eight heads of one token, eight lanes a head: lane c of them
// holds dims 8c .. 8c+7 and 64+8c .. 64+8c+7, the two halves of eight
// rotation pairs, in two 16-byte loads.
__global__ __launch_bounds__(256) void qk_pages_kernel(QkArgs a)
{
    const int heads = a.n_heads + 2 * a.n_kv, blocks = (heads + 7) / 8;
    const long unit = (long)blockIdx.x * 4 + threadIdx.x / 64;
    const int t = (int)(unit / blocks), lane = threadIdx.x & 63, c = lane & 7;
    const int h = (int)(unit % blocks) * 8 + lane / 8;
    if (t >= a.n_tok) return;
    const int pos = a.positions[t];
    if (pos < 0 || pos >= a.n_rope) return;
    const int64_t slot = a.slots[t];
    const bool live = h < heads, cached = slot >= 0 && slot < a.n_slots;
    float lo[8] = {}, hi[8] = {};
    if (live) {
        const uint16_t* row = a.qkv + t * a.qkv_stride + (size_t)h * kHeadDim;
        unpack8(ldg16u(row + 8 * c), lo);
        unpack8(ldg16u(row + 64 + 8 * c), hi);
    }
    if (h < a.n_heads + a.n_kv) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(lo[i], lo[i], __builtin_fmaf(hi[i], hi[i], ss));
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor(ss, m);
        const float r = 1.0f / __fsqrt_rn(ss * (1.0f / kHeadDim) + a.eps);
        const uint16_t* gamma = h < a.n_heads ? a.q_gamma : a.k_gamma;
        float g_lo[8], g_hi[8];
        unpack8(ldg16u(gamma + 8 * c), g_lo);
        unpack8(ldg16u(gamma + 64 + 8 * c), g_hi);
        const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * kHeadDim + 16 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 w = cs[i];
            const float cc[2] = {w.x, w.z}, sn[2] = {w.y, w.w};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int e = 2 * i + j;
                const float x = g_lo[e] * (lo[e] * r), y = g_hi[e] * (hi[e] * r);
                lo[e] = x * cc[j] - y * sn[j];
                hi[e] = y * cc[j] + x * sn[j];
            }
        }
    }
    if (!live) return;
    if (h < a.n_heads) {
        uint16_t* out = a.q_out + t * a.q_stride + (size_t)h * kHeadDim + 8 * c;
        *reinterpret_cast<uint4*>(out) = make_uint4(pack2_bf16(lo[0], lo[1]), pack2_bf16(lo[2], lo[3]),
                                                    pack2_bf16(lo[4], lo[5]), pack2_bf16(lo[6], lo[7]));
        *reinterpret_cast<uint4*>(out + 64) = make_uint4(pack2_bf16(hi[0], hi[1]), pack2_bf16(hi[2], hi[3]),
                                                         pack2_bf16(hi[4], hi[5]), pack2_bf16(hi[6], hi[7]));
        return;
    }
    if (!cached) return;
    const int e = h - a.n_heads;                       // k heads, then v heads
    const uint2 w_lo = codes8(lo, a.kv_inv[e]), w_hi = codes8(hi, a.kv_inv[e]);
    const int64_t page = slot / kPage;
    const int key = (int)(slot % kPage);
    if (e < a.n_kv) {
        uint8_t* p = a.k_pages + (size_t)(page * a.n_kv + e) * kPageBytes;
        *reinterpret_cast<uint2*>(p + k_byte(key, 8 * c)) = w_lo;
        *reinterpret_cast<uint2*>(p + k_byte(key, 64 + 8 * c)) = w_hi;
    } else {
        uint8_t* p = a.v_pages + (size_t)(page * a.n_kv + e - a.n_kv) * kPageBytes;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[v_byte(key, 8 * c + i)] = (uint8_t)((i < 4 ? w_lo.x : w_lo.y) >> (8 * (i & 3)));
            p[v_byte(key, 64 + 8 * c + i)] = (uint8_t)((i < 4 ? w_hi.x : w_hi.y) >> (8 * (i & 3)));
        }
    }
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
    if (!heads_ok(n_heads, n_kv_heads, head_dim) || n_tok < 1 || n_pages < 1 || n_rope_pos < 1 ||
        q_stride < (int64_t)n_heads * kHeadDim || qkv_stride < heads * kHeadDim)
        return HEPH_ERR_SHAPE;
    if (!aligned(q_out_bf16, 16) || !aligned(qkv_bf16, 16) || !aligned(q_gamma, 16) ||
        !aligned(k_gamma, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
        !aligned(rope_table, 16) || q_stride % 8 || qkv_stride % 8)
        return HEPH_ERR_ALIGN;
    // in place only with the rows where they are: another stride would let one
    // wave overwrite what the next one reads
    if (q_out_bf16 == qkv_bf16 && q_stride != qkv_stride) return HEPH_ERR_SHAPE;
    const int64_t units = (int64_t)n_tok * ((heads + 7) / 8), blocks = (units + 3) / 4;
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
    qk_pages_kernel<<<(unsigned)blocks, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
