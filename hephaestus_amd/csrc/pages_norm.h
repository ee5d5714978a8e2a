// pages_norm.h - RMSNorm and rotation of one head, eight lanes a head, for the ops that
// write the paged cache.
#pragma once

#include "pages.h"

namespace heph {

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

// Lane c of eight: dims 8c .. 8c+7 (lo) and 64+8c .. 64+8c+7 (hi) of a head, the two halves of
// eight rotation pairs, normalized, times gamma and rotated by w, its (cos, sin) pairs. All eight
// lanes call it.
__device__ __forceinline__ void norm_rope(float (&lo)[8], float (&hi)[8], const uint4& x_lo, const uint4& x_hi,
                                          const uint4& y_lo, const uint4& y_hi, const float4 (&w)[4], float eps)
{
    float g_lo[8], g_hi[8];
    unpack8(x_lo, lo);
    unpack8(x_hi, hi);
    unpack8(y_lo, g_lo);
    unpack8(y_hi, g_hi);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(lo[i], lo[i], __builtin_fmaf(hi[i], hi[i], ss));
    // over the eight lanes: the neighbour, the other pair, the other quad (whose lanes are equal by then)
    auto other = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    ss += other(ss, std::integral_constant<int, 0xB1>{});
    ss += other(ss, std::integral_constant<int, 0x4E>{});
    ss += other(ss, std::integral_constant<int, 0x141>{});
    const float r = 1.0f / __fsqrt_rn(ss * (1.0f / kHeadDim) + eps);
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
}

// A store past the caches (nontemporal): for long streams.
__device__ __forceinline__ void store_past(uint16_t* p, const uint4& x)
{
    __builtin_nontemporal_store(i32x4{(int)x.x, (int)x.y, (int)x.z, (int)x.w}, reinterpret_cast<i32x4*>(p));
}

// Such a lane's values to its head at out, as bf16; PAST: past the caches.
template <bool PAST = false>
__device__ __forceinline__ void store_head(uint16_t* out, const float (&lo)[8], const float (&hi)[8])
{
    const uint4 a = make_uint4(pack2_bf16(lo[0], lo[1]), pack2_bf16(lo[2], lo[3]), pack2_bf16(lo[4], lo[5]),
                               pack2_bf16(lo[6], lo[7]));
    const uint4 b = make_uint4(pack2_bf16(hi[0], hi[1]), pack2_bf16(hi[2], hi[3]), pack2_bf16(hi[4], hi[5]),
                               pack2_bf16(hi[6], hi[7]));
    if constexpr (PAST) {
        store_past(out, a);
        store_past(out + 64, b);
    } else {
        *reinterpret_cast<uint4*>(out) = a;
        *reinterpret_cast<uint4*>(out + 64) = b;
    }
}

}  // namespace heph
