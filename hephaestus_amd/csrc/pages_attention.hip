// pages_attention.hip - attention of a batch over the paged E4M3 cache.
#include "pages.h"

namespace heph {
namespace {

constexpr int kMagic = 0x41505031;
struct PlanHeader {
    int magic, n_tok, n_seqs, n_groups, table_pages, n_heads, n_kv, pad;
};

// Per token: its sequence (-1: none) and how many keys it attends to.
__global__ __launch_bounds__(256) void plan_kernel(PlanHeader* plan, PlanHeader h,
                                                   const int32_t* q_start, const int32_t* kv_len)
{
    int2* tok = reinterpret_cast<int2*>(plan + 1);
    for (int t = threadIdx.x; t < h.n_tok; t += 256) {
        int seq = -1, limit = 0, start = 0;
        for (int s = 0; s < h.n_seqs; ++s) {
            start = min(max(q_start[s], start), h.n_tok);
            const int end = min(max(q_start[s + 1], start), h.n_tok);
            if (t >= start && t < end) {
                seq = s;
                limit = min(max(kv_len[s], 0), h.table_pages * kPage) - (end - start) + (t - start) + 1;
            }
        }
        tok[t] = make_int2(seq, max(limit, 0));
    }
    if (threadIdx.x == 0) *plan = h;
}

struct AttnArgs {
    uint16_t* out;
    const uint16_t* q;
    int64_t q_stride;
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    const float* kv_scale;
    const int32_t* table;
    const PlanHeader* plan;
    int n_pages, table_pages, n_tok, n_seqs, n_groups, n_heads, n_kv;
};

__device__ __forceinline__ float e4m3_float(uint32_t w, int i)
{
    const uint32_t c = w >> (8 * i) & 0xFF;
    return __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false)[0];
}

// One wave per (token, head), one key a lane: scores and running maximum and
// sum page by page, then two dims a lane of the product with V.
__global__ __launch_bounds__(64) void attention_kernel(AttnArgs a)
{
    __shared__ float q[kHeadDim], prob[kPage];
    const PlanHeader h = *a.plan;
    if (h.magic != kMagic || h.n_tok != a.n_tok || h.n_seqs != a.n_seqs ||
        h.n_groups != a.n_groups || h.table_pages != a.table_pages || h.n_heads != a.n_heads ||
        h.n_kv != a.n_kv)
        return;
    const int t = blockIdx.x, head = blockIdx.y, kv = head / (a.n_heads / a.n_kv), l = threadIdx.x;
    const int2 tok = reinterpret_cast<const int2*>(a.plan + 1)[t];
    if (tok.x < 0) return;
    for (int d = l; d < kHeadDim; d += 64)
        q[d] = bf16_value(a.q[t * a.q_stride + (size_t)head * kHeadDim + d]);
    const float scale = a.kv_scale[kv] * 0.08838834764831845f;
    float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    __syncthreads();
    for (int p = 0; p * kPage < tok.y; ++p) {
        const int id = a.table[(size_t)tok.x * a.table_pages + p];
        if (id < 0 || id >= a.n_pages) continue;
        const uint8_t* kp = a.k_pages + ((size_t)id * a.n_kv + kv) * kPageBytes;
        const uint8_t* vp = a.v_pages + ((size_t)id * a.n_kv + kv) * kPageBytes;
        const bool seen = p * kPage + l < tok.y;
        float s = 0.0f;
        for (int d = 0; d < kHeadDim; d += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kp + k_byte(l, d));
            for (int i = 0; i < 4; ++i) s = __builtin_fmaf(q[d + i], e4m3_float(w, i), s);
        }
        s = seen ? s * scale : -INFINITY;
        const float mp = fmaxf(m, wave_fold_max64(s)), base = mp == -INFINITY ? 0.0f : mp;
        const float e = seen ? __expf(s - base) : 0.0f, f = __expf(m - base);
        __syncthreads();
        prob[v_place(l)] = e;
        __syncthreads();
        sum = sum * f + wave_fold_sum64(e);
        o0 *= f;
        o1 *= f;
        const unsigned long long mask = __ballot(seen);
        for (int j = 0; j < kPage; ++j) {
            if (!(mask >> j & 1)) break;
            const float pj = prob[v_place(j)];
            o0 = __builtin_fmaf(pj, e4m3_float(vp[v_byte(j, l)], 0), o0);
            o1 = __builtin_fmaf(pj, e4m3_float(vp[v_byte(j, l + 64)], 0), o1);
        }
        m = mp;
    }
    const float f = sum == 0.0f && m == -INFINITY ? 0.0f : a.kv_scale[a.n_kv + kv] / sum;
    uint16_t* out = a.out + ((size_t)t * a.n_heads + head) * kHeadDim;
    out[l] = f32_to_bf16(o0 * f);
    out[l + 64] = f32_to_bf16(o1 * f);
}

bool sizes_ok(int n_tok, int n_seqs, int n_groups, int n_heads, int n_kv)
{
    return heads_ok(n_heads, n_kv, kHeadDim) && n_tok >= 1 && n_seqs >= 1 && n_groups >= 0 &&
           n_groups <= n_seqs && n_tok <= (1 << 20) && n_seqs <= (1 << 16) && n_heads <= 4096;
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

size_t heph_pages_attention_plan_bytes(int n_tok, int n_seqs, int n_groups, int n_heads,
                                       int n_kv_heads)
{
    if (!sizes_ok(n_tok, n_seqs, n_groups, n_heads, n_kv_heads)) return 0;
    return sizeof(PlanHeader) + sizeof(int2) * (size_t)n_tok;
}

size_t heph_pages_attention_ws_bytes(int n_tok, int n_seqs, int n_groups, int n_heads,
                                     int n_kv_heads)
{
    if (!sizes_ok(n_tok, n_seqs, n_groups, n_heads, n_kv_heads)) return 0;
    return 16;
}

int heph_pages_attention_plan(void* plan, size_t plan_bytes, const int32_t* q_start,
                              const int32_t* kv_len, const int32_t* group_start,
                              const int32_t* shared_pages, int n_tok, int n_seqs, int n_groups,
                              int table_pages, int n_heads, int n_kv_heads, void* stream)
{
    if (!plan || !q_start || !kv_len || (n_groups > 0 && (!group_start || !shared_pages)))
        return HEPH_ERR_NULL;
    if (!sizes_ok(n_tok, n_seqs, n_groups, n_heads, n_kv_heads) || table_pages < 1 ||
        table_pages > HEPH_ATTN_MAX_KEYS / kPage)
        return HEPH_ERR_SHAPE;
    if (!aligned(plan, 16)) return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_pages_attention_plan_bytes(n_tok, n_seqs, n_groups, n_heads, n_kv_heads))
        return HEPH_ERR_WORKSPACE;
    if (int st = check_device()) return st;
    const PlanHeader h{kMagic, n_tok, n_seqs, n_groups, table_pages, n_heads, n_kv_heads, 0};
    plan_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(static_cast<PlanHeader*>(plan), h,
                                                                 q_start, kv_len);
    return status_of(hipGetLastError());
}

int heph_pages_attention(void* out_bf16, const void* q_bf16, int64_t q_stride,
                         const uint8_t* k_pages, const uint8_t* v_pages, int n_pages,
                         const float* kv_scale, const int32_t* page_table, int table_pages,
                         const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes,
                         int n_tok, int n_seqs, int n_groups, int n_heads, int n_kv_heads,
                         int head_dim, void* stream)
{
    if (!out_bf16 || !q_bf16 || !k_pages || !v_pages || !kv_scale || !page_table || !plan || !ws)
        return HEPH_ERR_NULL;
    if (head_dim != kHeadDim || !sizes_ok(n_tok, n_seqs, n_groups, n_heads, n_kv_heads) ||
        n_pages < 1 || table_pages < 1 || table_pages > HEPH_ATTN_MAX_KEYS / kPage ||
        q_stride < (int64_t)n_heads * kHeadDim)
        return HEPH_ERR_SHAPE;
    if (!aligned(out_bf16, 16) || !aligned(q_bf16, 16) || !aligned(k_pages, 16) ||
        !aligned(v_pages, 16) || !aligned(plan, 16) || !aligned(ws, 16) || q_stride % 8)
        return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_pages_attention_plan_bytes(n_tok, n_seqs, n_groups, n_heads, n_kv_heads) ||
        ws_bytes < heph_pages_attention_ws_bytes(n_tok, n_seqs, n_groups, n_heads, n_kv_heads))
        return HEPH_ERR_WORKSPACE;
    if (int st = check_device()) return st;
    AttnArgs a;
    a.out = static_cast<uint16_t*>(out_bf16);
    a.q = static_cast<const uint16_t*>(q_bf16);
    a.q_stride = q_stride;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.kv_scale = kv_scale;
    a.table = page_table;
    a.plan = static_cast<const PlanHeader*>(plan);
    a.n_pages = n_pages;
    a.table_pages = table_pages;
    a.n_tok = n_tok;
    a.n_seqs = n_seqs;
    a.n_groups = n_groups;
    a.n_heads = n_heads;
    a.n_kv = n_kv_heads;
    attention_kernel<<<dim3(n_tok, n_heads), 64, 0, static_cast<hipStream_t>(stream)>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
