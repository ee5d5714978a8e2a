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

// s_waitcnt: at most N of this wave's vector memory operations and no LDS one left.
template <int N>
__device__ __forceinline__ void wait_vm()
{
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

// LDS accesses of the workgroup before and behind it are ordered; loads from
// memory stay in flight (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

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
