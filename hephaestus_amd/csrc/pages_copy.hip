// pages_copy.hip - copies of pages within the pools of the paged KV cache.
#include <algorithm>
#include <new>
#include <vector>

#include "pages.h"

namespace heph {
namespace {

// The pairs travel in the launch's arguments: no upload, and a captured launch
// keeps them.
constexpr int kPairs = 256;
struct CopyArgs {
    uint8_t* pool[2];
    float* scale;                  // [n_layers][n_pages][2 * n_kv], or NULL
    size_t page_bytes, layer_bytes;
    int n_kv, n_pages;
    int src[kPairs], dst[kPairs];
};

// One workgroup moves one kv head of one page, two loads of 16 bytes a thread. Bound by
// memory: 64 pages of 36 layers, 8 kv heads (604 MB read and written) in 115 us, 5.25 TB/s,
// what a large copy reaches.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a)
{
    const int head = blockIdx.x % a.n_kv, pair = blockIdx.x / a.n_kv;
    uint8_t* pool = a.pool[blockIdx.z] + (size_t)blockIdx.y * a.layer_bytes + (size_t)head * kPageBytes;
    const uint8_t* from = pool + (size_t)a.src[pair] * a.page_bytes;
    uint8_t* to = pool + (size_t)a.dst[pair] * a.page_bytes;
    const int o = threadIdx.x * 16;
    const uint4 x = ldg16u(from + o), y = ldg16u(from + o + 4096);
    *reinterpret_cast<uint4*>(to + o) = x;
    *reinterpret_cast<uint4*>(to + o + 4096) = y;
    if (a.scale && threadIdx.x == 0) {             // the block's scale
        float* s = a.scale + ((size_t)blockIdx.y * a.n_pages * 2 + blockIdx.z) * a.n_kv + head;
        s[(size_t)a.dst[pair] * 2 * a.n_kv] = s[(size_t)a.src[pair] * 2 * a.n_kv];
    }
}

}  // namespace
}  // namespace heph

using namespace heph;

static int copy_pages(uint8_t* k_pages, uint8_t* v_pages, float* scale, int n_layers, int n_pages,
                      int n_kv_heads, const int32_t* src, const int32_t* dst, int n, void* stream)
{
    if (!k_pages || !v_pages || (n > 0 && (!src || !dst))) return HEPH_ERR_NULL;
    if (n_layers < 1 || n_layers > 65535 || n_pages < 1 || n_kv_heads < 1 || n_kv_heads > 4096 ||
        n < 0 || n > n_pages)
        return HEPH_ERR_SHAPE;
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(scale, 4)) return HEPH_ERR_ALIGN;
    if (n == 0) return HEPH_OK;
    try {
        // destinations that repeat or are read by another pair would race
        std::vector<int32_t> to(dst, dst + n);
        std::sort(to.begin(), to.end());
        if (to.front() < 0 || to.back() >= n_pages ||
            std::adjacent_find(to.begin(), to.end()) != to.end())
            return HEPH_ERR_SHAPE;
        for (int i = 0; i < n; ++i)
            if (src[i] < 0 || src[i] >= n_pages ||
                std::binary_search(to.begin(), to.end(), src[i]))
                return HEPH_ERR_SHAPE;
    } catch (const std::bad_alloc&) {
        return HEPH_ERR_SCRATCH;
    }
    if (int st = check_device()) return st;
    CopyArgs a;
    a.pool[0] = k_pages;
    a.pool[1] = v_pages;
    a.page_bytes = (size_t)n_kv_heads * kPageBytes;
    a.layer_bytes = (size_t)n_pages * a.page_bytes;
    a.n_kv = n_kv_heads;
    a.n_pages = n_pages;
    a.scale = scale;
    for (int i = 0; i < n; i += kPairs) {
        const int pairs = std::min(kPairs, n - i);
        std::copy(src + i, src + i + pairs, a.src);
        std::copy(dst + i, dst + i + pairs, a.dst);
        copy_pages_kernel<<<dim3((unsigned)n_kv_heads * pairs, n_layers, 2), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
        if (hipGetLastError() != hipSuccess) return HEPH_ERR_LAUNCH;
    }
    return HEPH_OK;
}

extern "C" {

int heph_copy_pages(uint8_t* k_pages, uint8_t* v_pages, int n_layers, int n_pages, int n_kv_heads,
                    const int32_t* src, const int32_t* dst, int n, void* stream)
{
    return copy_pages(k_pages, v_pages, nullptr, n_layers, n_pages, n_kv_heads, src, dst, n, stream);
}

int heph_copy_pages_scaled(uint8_t* k_pages, uint8_t* v_pages, float* page_scale, int n_layers,
                           int n_pages, int n_kv_heads, const int32_t* src, const int32_t* dst,
                           int n, void* stream)
{
    if (!page_scale) return HEPH_ERR_NULL;
    return copy_pages(k_pages, v_pages, page_scale, n_layers, n_pages, n_kv_heads, src, dst, n, stream);
}

}  // extern "C"
