// pages.h - the paged KV cache's layout (include/hephserve.h) and small device
// helpers of the serving ops.
#pragma once

#include "heph_kernels.h"
#include "../../include/hephserve.h"

namespace heph {

constexpr int kPage = HEPH_PAGE_KEYS;
constexpr int kHeadDim = 128;
constexpr int kPageBytes = kPage * kHeadDim;   // of one kv head in one pool

// Where key j of a page lies in its V rows.
__host__ __device__ __forceinline__ int v_place(int j)
{
    return (j / 4 % 4) * 16 + (j / 32) * 8 + (j / 16 % 2) * 4 + j % 4;
}

// Byte of key j, dim d within a page of one kv head.
__host__ __device__ __forceinline__ int k_byte(int j, int d) { return d / 64 * 4096 + j * 64 + d % 64; }
__host__ __device__ __forceinline__ int v_byte(int j, int d) { return d * 64 + v_place(j); }

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline int status_of(hipError_t e) { return e == hipSuccess ? HEPH_OK : HEPH_ERR_LAUNCH; }

// Query heads per kv head of the serving ops.
constexpr int kMaxGroup = 64;
inline bool heads_ok(int n_heads, int n_kv, int head_dim)
{
    return head_dim == kHeadDim && n_kv >= 1 && n_heads >= n_kv && n_heads % n_kv == 0 &&
           n_heads / n_kv <= kMaxGroup;
}

}  // namespace heph
