// lora.hip - low-rank adapters of many requests beside one projection:
// c = base + scale[i] (x a[i]^T) b[i]^T, row m with adapter i = ids[m].
//
// The plan kernel sorts the rows by adapter into tiles of 16 (decode) or 64 rows,
// so that an adapter's weights are read once a tile. Two launches follow:
//   shrink: t = x a^T, a workgroup per (tile, part of K), f32 partials
//   expand: c = base + (scale t) b^T, a workgroup per (tile, part of N)
// both on v_mfma_f32_16x16x32_bf16. t enters the second product as a bf16 and the
// bf16 of its remainder (16 bits of mantissa): the product has matrix cores to
// spare, as both launches are bound by what they stream.
#include <algorithm>

#include "pages.h"

namespace heph {
namespace {

constexpr int kMagic = 0x4C4F5242;
constexpr int kMaxAdapters = HEPH_LORA_MAX_ADAPTERS;
constexpr int kPlanThreads = 1024;

struct PlanHeader {
    int magic, m, n_adapters, n_tiles;
};
// Rows rows[start .. start + count) have the adapter (-1: none).
struct Tile {
    int adapter, start, count, pad;
};

// Rows of a tile: a decode batch has few of each adapter, a prompt's rows fill 64.
__host__ __device__ __forceinline__ int tile_rows(int M) { return M <= 256 ? 16 : 64; }
__host__ __device__ __forceinline__ int max_tiles(int M, int n_adapters)
{
    const int full = M / tile_rows(M) + n_adapters + 1;     // one short tile an adapter at most
    return full < M ? full : M;
}
__host__ __device__ inline Tile* plan_tiles(PlanHeader* p) { return reinterpret_cast<Tile*>(p + 1); }
__host__ __device__ inline int* plan_rows(PlanHeader* p, int M, int n_adapters)
{
    return reinterpret_cast<int*>(plan_tiles(p) + max_tiles(M, n_adapters));
}

// Counting sort of the rows by adapter. Rows of one adapter come in no fixed
// order; no result depends on it.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanHeader* plan, const int32_t* ids, int M,
                                                            int n_adapters)
{
    __shared__ int count[kMaxAdapters + 1], red[2][kPlanThreads / 64];
    const int t = threadIdx.x, nt = blockDim.x, groups = n_adapters + 1, TR = tile_rows(M);
    Tile* tiles = plan_tiles(plan);
    int* rows = plan_rows(plan, M, n_adapters);
    for (int g = t; g < groups; g += nt) count[g] = 0;
    __syncthreads();
    auto group_of = [&](int m) {
        const int id = ids[m];
        return id >= 0 && id < n_adapters ? id : n_adapters;         // none: the last group
    };
    for (int m = t; m < M; m += nt) atomicAdd(&count[group_of(m)], 1);
    __syncthreads();
    int row0 = 0, tile0 = 0;                                         // of the groups before
    for (int g0 = 0; g0 < groups; g0 += nt) {
        const int g = g0 + t, n = g < groups ? count[g] : 0, nTiles = (n + TR - 1) / TR;
        int row = n, tile = nTiles;
        for (int o = 1; o < 64; o <<= 1) {
            const int a = __shfl_up(row, o), b = __shfl_up(tile, o);
            if ((t & 63) >= o) {
                row += a;
                tile += b;
            }
        }
        if ((t & 63) == 63) {
            red[0][t / 64] = row;
            red[1][t / 64] = tile;
        }
        __syncthreads();
        int row_sum = 0, tile_sum = 0;
        for (int w = 0; w < nt / 64; ++w) {
            if (w < t / 64) {
                row += red[0][w];
                tile += red[1][w];
            }
            row_sum += red[0][w];
            tile_sum += red[1][w];
        }
        row += row0 - n;
        tile += tile0 - nTiles;
        for (int i = 0; i < nTiles; ++i)
            tiles[tile + i] = Tile{g < n_adapters ? g : -1, row + i * TR, min(TR, n - i * TR), 0};
        if (g < groups) count[g] = row;                              // now the group's next place
        row0 += row_sum;
        tile0 += tile_sum;
        __syncthreads();
    }
    for (int m = t; m < M; m += nt) rows[atomicAdd(&count[group_of(m)], 1)] = m;
    if (t == 0) *plan = PlanHeader{kMagic, M, n_adapters, tile0};
}

struct LoraArgs {
    void* c;
    const void* base;
    const uint16_t* x;
    const uint16_t* a;
    const uint16_t* b;
    const float* scale;
    PlanHeader* plan;
    float* part;             // [splits][M][r], rows in the plan's order
    int M, N, K, r, n_adapters, splits, n_chunk;
};

__device__ __forceinline__ bool plan_fits(const PlanHeader& h, const LoraArgs& g)
{
    return h.magic == kMagic && h.m == g.M && h.n_adapters == g.n_adapters;
}

__device__ __forceinline__ bf16x8 load8(const uint16_t* p, bool there)
{
    const i32x4 zero = {0, 0, 0, 0};
    return __builtin_bit_cast(bf16x8, there ? ldg16(p) : zero);
}

// Steps of 64 K: a lane holds 16 consecutive elements of a row of x and of a, two
// matrix instructions' worth (their order along K is the same on both sides).
constexpr int kStep = 64;

// RT 16-row tiles, RK 16-rank tiles. The workgroup's part of K goes in steps to its
// four waves, whose sums meet in LDS.
template <int RT, int RK>
__global__ __launch_bounds__(256) void shrink_kernel(LoraArgs g)
{
    __shared__ f32x4 lds[3][RT * RK][64];
    const PlanHeader h = *g.plan;
    const int tile = blockIdx.x / g.splits, split = blockIdx.x % g.splits;
    if (!plan_fits(h, g) || tile >= h.n_tiles) return;
    const Tile tl = plan_tiles(g.plan)[tile];
    if (tl.adapter < 0) return;
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, c = l & 15, g4 = l >> 4;
    const int steps = (g.K + kStep - 1) / kStep;
    const int s0 = (int)((long)steps * split / g.splits), s1 = (int)((long)steps * (split + 1) / g.splits);
    const int* rows = plan_rows(g.plan, g.M, g.n_adapters) + tl.start;
    const uint16_t *x[RT], *a[RK];
#pragma unroll
    for (int i = 0; i < RT; ++i)      // (rows past the tile's end: its last one again)
        x[i] = g.x + (size_t)rows[min(i * 16 + c, tl.count - 1)] * g.K + g4 * 16;
#pragma unroll
    for (int j = 0; j < RK; ++j)
        a[j] = g.a + ((size_t)tl.adapter * g.r + min(j * 16 + c, g.r - 1)) * g.K + g4 * 16;
    f32x4 acc[RT][RK];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < RK; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
#pragma unroll 2
    for (int s = s0 + wave; s < s1; s += 4) {
        const int k = s * kStep;
        const bool there = k + g4 * 16 < g.K;
        bf16x8 xs[RT][2], as[RK][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int j = 0; j < RK; ++j) as[j][e] = load8(a[j] + k + 8 * e, there);
#pragma unroll
            for (int i = 0; i < RT; ++i) xs[i][e] = load8(x[i] + k + 8 * e, there);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < RK; ++j) acc[i][j] = mfma_bf16(as[j][e], xs[i][e], acc[i][j]);
    }
    if (wave > 0)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < RK; ++j) lds[wave - 1][i * RK + j][l] = acc[i][j];
    __syncthreads();
    // lane: ranks 4 g4 .. of row c
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < RK; ++j) {
                const f32x4 v = ((acc[i][j] + lds[0][i * RK + j][l]) + lds[1][i * RK + j][l]) + lds[2][i * RK + j][l];
                const int row = i * 16 + c, rank = j * 16 + g4 * 4;
                if (row < tl.count && rank < g.r)
                    *reinterpret_cast<f32x4*>(g.part + ((size_t)split * g.M + tl.start + row) * g.r + rank) = v;
            }
}

// F operand pieces of 32 ranks (F = 0: 16 ranks, the remainders in the other half
// of one piece). Outputs transposed, b as the first operand with its rows in the
// order that leaves eight consecutive columns of a row in a lane.
template <int RT, int F, bool F32>
__global__ __launch_bounds__(256) void expand_kernel(LoraArgs g)
{
    constexpr int P = F == 0 ? 1 : F, PARTS = F == 0 ? 1 : 2;
    __shared__ bf16x8 lds[RT][P][PARTS][64];
    const PlanHeader h = *g.plan;
    const int chunks = (g.N + g.n_chunk - 1) / g.n_chunk;
    const int tile = blockIdx.x / chunks, n0 = blockIdx.x % chunks * g.n_chunk;
    if (!plan_fits(h, g) || tile >= h.n_tiles) return;
    const Tile tl = plan_tiles(g.plan)[tile];
    const bool copy = tl.adapter < 0;
    if (copy && g.c == g.base) return;
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, c = l & 15, g4 = l >> 4;
    if (!copy) {
        const float scale = g.scale[tl.adapter];
        for (int u = threadIdx.x; u < RT * P * 64; u += 256) {
            const int i = u / (P * 64), f = u / 64 % P, ul = u & 63, row = i * 16 + (ul & 15);
            const int rank = F == 0 ? (ul >> 4 & 1) * 8 : f * 32 + (ul >> 4) * 8;
            f32x4 s[2] = {};
            if (row < tl.count && rank < g.r) {
                const float* p = g.part + (size_t)(tl.start + row) * g.r + rank;
                for (int k = 0; k < g.splits; ++k, p += (size_t)g.M * g.r) {
                    s[0] += *reinterpret_cast<const f32x4*>(p);
                    s[1] += *reinterpret_cast<const f32x4*>(p + 4);
                }
            }
            bf16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = s[e / 4][e % 4] * scale;
                hi[e] = (__bf16)v;
                lo[e] = (__bf16)(v - (float)hi[e]);
            }
            if constexpr (F == 0) {
                lds[i][0][0][ul] = ul < 32 ? hi : lo;
            } else {
                lds[i][f][0][ul] = hi;
                lds[i][f][1][ul] = lo;
            }
        }
        __syncthreads();
    }
    bf16x8 t[RT][P][PARTS];
    int row[RT];
    const int* rows = plan_rows(g.plan, g.M, g.n_adapters) + tl.start;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        row[i] = i * 16 + c < tl.count ? rows[i * 16 + c] : -1;
#pragma unroll
        for (int f = 0; f < P; ++f)
#pragma unroll
            for (int e = 0; e < PARTS; ++e) t[i][f][e] = lds[i][f][e][l];
    }
    const uint16_t* b = g.b + (size_t)(copy ? 0 : tl.adapter) * g.N * g.r;
    const int n_end = min(n0 + g.n_chunk, g.N);
    for (int n = n0 + wave * 32; n < n_end; n += 128) {
        // this lane's eight columns are all inside N or all past it (N % 16 == 0)
        const int col = n + g4 * 8;
        const bool inside = col < g.N;
        f32x4 v[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            v[i][0] = v[i][1] = f32x4{0, 0, 0, 0};
            if (row[i] >= 0 && inside) {
                const size_t o = (size_t)row[i] * g.N + col;
                if constexpr (F32) {
                    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(g.base) + o);
                    v[i][0] = p[0];
                    v[i][1] = p[1];
                } else {
                    const uint4 w = ldg16u(static_cast<const uint16_t*>(g.base) + o);
                    v[i][0] = f32x4{bf16lo(w.x), bf16hi(w.x), bf16lo(w.y), bf16hi(w.y)};
                    v[i][1] = f32x4{bf16lo(w.z), bf16hi(w.z), bf16lo(w.w), bf16hi(w.w)};
                }
            }
        }
        if (!copy) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int bn = n + (c >> 2) * 8 + j * 4 + (c & 3);
                bf16x8 w[P];
#pragma unroll
                for (int f = 0; f < P; ++f) {
                    const int rank = F == 0 ? (g4 & 1) * 8 : f * 32 + g4 * 8;
                    w[f] = load8(b + (size_t)min(bn, g.N - 1) * g.r + rank, rank < g.r);
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    f32x4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int f = 0; f < P; ++f)
#pragma unroll
                        for (int e = PARTS - 1; e >= 0; --e) d = mfma_bf16(w[f], t[i][f][e], d);
                    v[i][j] += d;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (row[i] >= 0 && inside) {
                const size_t o = (size_t)row[i] * g.N + col;
                if constexpr (F32) {
                    f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(g.c) + o);
                    p[0] = v[i][0];
                    p[1] = v[i][1];
                } else {
                    auto two = [](float x, float y) { return (uint32_t)f32_to_bf16(x) | (uint32_t)f32_to_bf16(y) << 16; };
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.c) + o) =
                        make_uint4(two(v[i][0][0], v[i][0][1]), two(v[i][0][2], v[i][0][3]),
                                   two(v[i][1][0], v[i][1][1]), two(v[i][1][2], v[i][1][3]));
                }
            }
    }
}

bool sizes_ok(int M, int n_adapters)
{
    return M >= 1 && M <= (1 << 20) && n_adapters >= 1 && n_adapters <= kMaxAdapters;
}
bool rank_ok(int rank) { return rank >= 8 && rank <= 128 && rank % 8 == 0; }

// Parts of K: as many as fill the device twice over, each at least a step a wave.
int k_splits(int M, int n_adapters, int K)
{
    const int steps = (K + kStep - 1) / kStep, want = 2 * kPlanCUs / max_tiles(M, n_adapters);
    return std::max(1, std::min(std::min((steps + 3) / 4, want), 16));
}

template <int RT>
void launch_shrink(const LoraArgs& g, unsigned blocks, hipStream_t s)
{
    if (g.r <= 16) shrink_kernel<RT, 1><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 32) shrink_kernel<RT, 2><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 64) shrink_kernel<RT, 4><<<blocks, 256, 0, s>>>(g);
    else shrink_kernel<RT, 8><<<blocks, 256, 0, s>>>(g);
}

template <int RT, bool F32>
void launch_expand(const LoraArgs& g, unsigned blocks, hipStream_t s)
{
    if (g.r <= 16) expand_kernel<RT, 0, F32><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 32) expand_kernel<RT, 1, F32><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 64) expand_kernel<RT, 2, F32><<<blocks, 256, 0, s>>>(g);
    else expand_kernel<RT, 4, F32><<<blocks, 256, 0, s>>>(g);
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" {

size_t heph_lora_plan_bytes(int M, int n_adapters)
{
    if (!sizes_ok(M, n_adapters)) return 0;
    return sizeof(PlanHeader) + sizeof(Tile) * (size_t)max_tiles(M, n_adapters) + 4 * (size_t)M;
}

size_t heph_lora_ws_bytes(int M, int n_adapters, int K, int rank)
{
    if (!sizes_ok(M, n_adapters) || K < 16 || !rank_ok(rank)) return 0;
    return 4 * (size_t)k_splits(M, n_adapters, K) * M * rank;
}

int heph_lora_plan(void* plan, size_t plan_bytes, const int32_t* ids, int M, int n_adapters,
                   void* stream)
{
    if (!plan || !ids) return HEPH_ERR_NULL;
    if (!sizes_ok(M, n_adapters)) return HEPH_ERR_SHAPE;
    if (!aligned(plan, 16)) return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_lora_plan_bytes(M, n_adapters)) return HEPH_ERR_WORKSPACE;
    if (int st = check_device()) return st;
    const int threads = std::min(kPlanThreads, std::max(64, (std::max(M, n_adapters + 1) + 63) / 64 * 64));
    plan_kernel<<<1, threads, 0, static_cast<hipStream_t>(stream)>>>(static_cast<PlanHeader*>(plan), ids, M,
                                                                     n_adapters);
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
    const int tiles = max_tiles(M, n_adapters), splits = k_splits(M, n_adapters, K);
    // columns a workgroup: more where that still leaves work for the device
    const int n_chunk = (long)tiles * N >= 512L * 4 * kPlanCUs ? 512 : 128;
    const int64_t expand = (int64_t)tiles * ((N + n_chunk - 1) / n_chunk);
    if (expand > INT32_MAX) return HEPH_ERR_UNSUPPORTED;
    if (int st = check_device()) return st;
    const LoraArgs g{c, base, x_bf16, a_bf16, b_bf16, scale,
                     static_cast<PlanHeader*>(const_cast<void*>(plan)), static_cast<float*>(ws), M, N, K,
                     rank, n_adapters, splits, n_chunk};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = c_dtype == HEPH_DTYPE_F32;
    if (tile_rows(M) == 16) {
        launch_shrink<1>(g, (unsigned)(tiles * splits), s);
        f32 ? launch_expand<1, true>(g, (unsigned)expand, s) : launch_expand<1, false>(g, (unsigned)expand, s);
    } else {
        launch_shrink<4>(g, (unsigned)(tiles * splits), s);
        f32 ? launch_expand<4, true>(g, (unsigned)expand, s) : launch_expand<4, false>(g, (unsigned)expand, s);
    }
    return status_of(hipGetLastError());
}

}  // extern "C"
