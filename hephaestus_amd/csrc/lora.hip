// lora.hip - low-rank adapters of many requests beside one projection.
#include "pages.h"

namespace heph {
namespace {

constexpr int kMagic = 0x4C4F5241;
struct PlanHeader {
    int magic, m, n_adapters, pad;
};

// Per row its adapter, -1 for none.
__global__ __launch_bounds__(256) void plan_kernel(PlanHeader* plan, PlanHeader h, const int32_t* ids)
{
    int* row = reinterpret_cast<int*>(plan + 1);
    for (int m = threadIdx.x; m < h.m; m += 256) {
        const int id = ids[m];
        row[m] = id >= 0 && id < h.n_adapters ? id : -1;
    }
    if (threadIdx.x == 0) *plan = h;
}

struct LoraArgs {
    void* c;
    const void* base;
    const uint16_t* x;
    const uint16_t* a;
    const uint16_t* b;
    const float* scale;
    const PlanHeader* plan;
    float* t;
    int M, N, K, r, n_adapters;
};

// t[m, j] = scale * x[m] . a[j]: one wave per (row, j).
__global__ __launch_bounds__(64) void shrink_kernel(LoraArgs g)
{
    if (g.plan->magic != kMagic || g.plan->m != g.M || g.plan->n_adapters != g.n_adapters) return;
    const int m = blockIdx.x, j = blockIdx.y;
    const int id = reinterpret_cast<const int*>(g.plan + 1)[m];
    if (id < 0) return;
    const uint16_t* x = g.x + (size_t)m * g.K;
    const uint16_t* w = g.a + ((size_t)id * g.r + j) * g.K;
    float s = 0.0f;
    for (int k = threadIdx.x; k < g.K; k += 64) s = __builtin_fmaf(bf16_value(x[k]), bf16_value(w[k]), s);
    s = wave_fold_sum64(s);
    if (threadIdx.x == 0) g.t[(size_t)m * g.r + j] = s * g.scale[id];
}

template <bool F32>
__global__ __launch_bounds__(256) void expand_kernel(LoraArgs g)
{
    if (g.plan->magic != kMagic || g.plan->m != g.M || g.plan->n_adapters != g.n_adapters) return;
    const int m = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x;
    if (n >= g.N) return;
    const int id = reinterpret_cast<const int*>(g.plan + 1)[m];
    const size_t o = (size_t)m * g.N + n;
    float s = F32 ? static_cast<const float*>(g.base)[o]
                  : bf16_value(static_cast<const uint16_t*>(g.base)[o]);
    if (id >= 0) {
        const uint16_t* w = g.b + ((size_t)id * g.N + n) * g.r;
        float d = 0.0f;
        for (int j = 0; j < g.r; ++j) d = __builtin_fmaf(g.t[(size_t)m * g.r + j], bf16_value(w[j]), d);
        s += d;
    }
    if constexpr (F32) static_cast<float*>(g.c)[o] = s;
    else static_cast<uint16_t*>(g.c)[o] = f32_to_bf16(s);
}

bool sizes_ok(int M, int n_adapters)
{
    return M >= 1 && M <= (1 << 20) && n_adapters >= 1 && n_adapters <= (1 << 16);
}
bool rank_ok(int rank) { return rank >= 8 && rank <= 128 && rank % 8 == 0; }

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

size_t heph_lora_plan_bytes(int M, int n_adapters)
{
    return sizes_ok(M, n_adapters) ? sizeof(PlanHeader) + 4 * (size_t)M : 0;
}

size_t heph_lora_ws_bytes(int M, int n_adapters, int K, int rank)
{
    return sizes_ok(M, n_adapters) && K >= 16 && rank_ok(rank) ? 4 * (size_t)M * rank : 0;
}

int heph_lora_plan(void* plan, size_t plan_bytes, const int32_t* ids, int M, int n_adapters,
                   void* stream)
{
    if (!plan || !ids) return HEPH_ERR_NULL;
    if (!sizes_ok(M, n_adapters)) return HEPH_ERR_SHAPE;
    if (!aligned(plan, 16)) return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_lora_plan_bytes(M, n_adapters)) return HEPH_ERR_WORKSPACE;
    if (int st = check_device()) return st;
    plan_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<PlanHeader*>(plan), PlanHeader{kMagic, M, n_adapters, 0}, ids);
    return status_of(hipGetLastError());
}

int heph_lora_add(void* c, int c_dtype, const void* base, const uint16_t* x_bf16,
                  const uint16_t* a_bf16, const uint16_t* b_bf16, const float* scale,
                  const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes, int M, int N,
                  int K, int rank, int n_adapters, void* stream)
{
    if (!c || !base || !x_bf16 || !a_bf16 || !b_bf16 || !scale || !plan || !ws) return HEPH_ERR_NULL;
    if (!sizes_ok(M, n_adapters) || !rank_ok(rank) || N < 16 || N % 16 || K < 16 || K % 16 ||
        N > (1 << 24) || K > (1 << 24))
        return HEPH_ERR_SHAPE;
    if (c_dtype != HEPH_DTYPE_BF16 && c_dtype != HEPH_DTYPE_F32) return HEPH_ERR_DTYPE;
    if (!aligned(c, 16) || !aligned(base, 16) || !aligned(x_bf16, 16) || !aligned(a_bf16, 16) ||
        !aligned(b_bf16, 16) || !aligned(plan, 16) || !aligned(ws, 16))
        return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_lora_plan_bytes(M, n_adapters) ||
        ws_bytes < heph_lora_ws_bytes(M, n_adapters, K, rank))
        return HEPH_ERR_WORKSPACE;
    if (int st = check_device()) return st;
    const LoraArgs g{c, base, x_bf16, a_bf16, b_bf16, scale, static_cast<const PlanHeader*>(plan),
                     static_cast<float*>(ws), M, N, K, rank, n_adapters};
    hipStream_t s = static_cast<hipStream_t>(stream);
    shrink_kernel<<<dim3(M, rank), 64, 0, s>>>(g);
    const dim3 grid(M, (N + 255) / 256);
    if (c_dtype == HEPH_DTYPE_F32) expand_kernel<true><<<grid, 256, 0, s>>>(g);
    else expand_kernel<false><<<grid, 256, 0, s>>>(g);
    return status_of(hipGetLastError());
}

}  // extern "C"
