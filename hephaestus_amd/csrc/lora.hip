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
//
// Measured (rank 16 unless said): 5 rows of 3 adapters, 2560 -> 6144 6.9 us, two launches
// of a chain of four loads each; 64 rows that use 32 of 40 adapters, 2560 -> 19456, 28 MB,
// 14.6 us (1.9 TB/s), 11.4 replayed on the same buffers, which the last-level cache holds;
// 4090 rows, 9728 -> 2560, rank 64, 41 us (123 MB, 3.0 TB/s), in f32 46. One launch for both
// products, each workgroup with all of t for itself, was slower throughout.
#include <algorithm>
#include <type_traits>

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

// Rows of a tile: a decode batch has few of each adapter, a prompt's rows fill 64. Tiles of
// 16 and of 64 rows, us (2560 -> 6144 of rank 16; 9728 -> 2560 of rank 64): 128 rows of 8
// adapters 8.2, 9.3; 12, 14. 256 of 40 9.8, 15; 21, 24. 512 of 8 9.4, 12; 20, 24. 1000 of 8
// 15, 16; 29, 25. 2000 of 40 26, 21; 62, 31. 2000 of 200 25, 32; 82, 83. The tiles of
// 16 win up to about 700 rows, with few rows of each adapter further still: the line lies
// lower than it could, at the longest decode batch that they were built for.
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

// Counting sort of the rows by adapter in one workgroup, once a step: 2.8 us for 64 rows,
// 6.2 for 4090 (two passes over the ids). Rows of one adapter come in no fixed order; no
// result depends on it.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanHeader* plan, const int32_t* ids, int M,
                                                            int n_adapters)
{
    __shared__ int count[kMaxAdapters + 1], red[2][kPlanThreads / 64];
    const int t = threadIdx.x, nt = blockDim.x, groups = n_adapters + 1, TR = tile_rows(M);
    Tile* tiles = plan_tiles(plan);
    int* rows = plan_rows(plan, M, n_adapters);
    for (int g = t; g < groups; g += nt) count[g] = 0;
    __syncthreads();
    // A place in the row's group. A prompt's neighbours share an adapter: one atomic for
    // a wave of them instead of 64 on one address.
    auto place = [&](int g) -> int {
        if (__all(g == __builtin_amdgcn_readfirstlane(g))) {
            const unsigned long long here = __ballot(1);
            int at = 0;
            if ((t & 63) == __ffsll((long long)here) - 1) at = atomicAdd(&count[g], __popcll(here));
            return __builtin_amdgcn_readfirstlane(at) +
                   __popcll(here & ((1ull << (t & 63)) - 1));
        }
        return atomicAdd(&count[g], 1);
    };
    // f(m, its group) for this thread's rows, four ids' loads at a time
    auto each_row = [&](auto f) {
        for (int m0 = t; m0 < M; m0 += 4 * nt) {
            int id[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) id[i] = ids[min(m0 + i * nt, M - 1)];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (m0 + i * nt < M)                                 // (none: the last group)
                    f(m0 + i * nt, id[i] >= 0 && id[i] < n_adapters ? id[i] : n_adapters);
        }
    };
    each_row([&](int, int g) { place(g); });
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
    each_row([&](int m, int g) { rows[place(g)] = m; });
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
    int M, N, K, r, n_adapters, splits, n_chunk, xcds;
};

__device__ __forceinline__ bool plan_fits(const PlanHeader& h, const LoraArgs& g)
{
    return h.magic == kMagic && h.m == g.M && h.n_adapters == g.n_adapters;
}

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) { return __builtin_bit_cast(bf16x8, ldg16(p)); }
__device__ __forceinline__ bf16x8 zero_unless(bf16x8 x, bool there)
{
    const i32x4 w = __builtin_bit_cast(i32x4, x), zero = {0, 0, 0, 0};
    return __builtin_bit_cast(bf16x8, there ? w : zero);
}

// s_waitcnt: at most N of this wave's vector memory operations and no LDS one left.
template <int N>
__device__ __forceinline__ void wait_vm()
{
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}
// The wait for a step with `left` later steps of P operations on their way.
template <int P, int MAX>
__device__ __forceinline__ void wait_steps(int left)
{
    if constexpr (MAX == 0) {
        wait_vm<0>();
    } else {
        if (left >= MAX) wait_vm<MAX * P>();
        else wait_steps<P, MAX - 1>(left);
    }
}
__device__ __forceinline__ void stage_barrier() { asm volatile("s_barrier" ::: "memory"); }

// Workgroups go to the XCDs in turn. With tiles for all of them (xcds = 8) a tile's parts
// all go to one, in both launches, so that t's parts are read through the L2 that wrote
// them and a tile's x, a and b stay in one L2; with few tiles (xcds = 1) they spread.
constexpr int kXcds = 8;
inline int xcds_for(int tiles) { return tiles >= 8 * kXcds ? kXcds : 1; }
inline int64_t blocks_for(int tiles, int parts)
{
    const int x = xcds_for(tiles);
    return (int64_t)((tiles + x - 1) / x * x) * parts;
}
__device__ __forceinline__ void tile_and_part(int xcds, int parts, int& tile, int& part)
{
    const int k = blockIdx.x / xcds;
    tile = k / parts * xcds + blockIdx.x % xcds;
    part = k % parts;
}

// K goes in steps of 64: two matrix instructions, 64 bytes of a row in each load.
constexpr int kStep = 64;

// Decode tiles: four waves take every fourth step of the workgroup's part of K, and
// their sums meet in LDS; RK tiles of 16 ranks. Bound by the stream of a, and by the
// latency of the loads in front of it.
template <int RK>
__global__ __launch_bounds__(256) void shrink_kernel(LoraArgs g)
{
    __shared__ f32x4 lds[3][RK][64];
    const PlanHeader h = *g.plan;
    int tile, split;
    tile_and_part(g.xcds, g.splits, tile, split);
    if (!plan_fits(h, g) || tile >= h.n_tiles) return;
    const Tile tl = plan_tiles(g.plan)[tile];
    if (tl.adapter < 0) return;
    const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (g.K + kStep - 1) / kStep;
    const int s0 = (int)((long)steps * split / g.splits), s1 = (int)((long)steps * (split + 1) / g.splits);
    // (rows past the tile's end: its last one again)
    const int row = plan_rows(g.plan, g.M, g.n_adapters)[tl.start + min(c, tl.count - 1)];
    const uint16_t *x = g.x + (size_t)row * g.K, *a[RK];
#pragma unroll
    for (int j = 0; j < RK; ++j)
        a[j] = g.a + ((size_t)tl.adapter * g.r + min(j * 16 + c, g.r - 1)) * g.K;
    f32x4 acc[RK];
#pragma unroll
    for (int j = 0; j < RK; ++j) acc[j] = f32x4{0, 0, 0, 0};
    for (int s = s0 + wave; s < s1; s += 4) {
        bf16x8 xs[2], as[RK][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // a piece past K: the row's end again, dropped below
            const int k = s * kStep + e * 32 + g4 * 8, at = min(k, g.K - 8);
            xs[e] = load8(x + at);
#pragma unroll
            for (int j = 0; j < RK; ++j) as[j][e] = load8(a[j] + at);
        }
        if (s * kStep + kStep > g.K)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool there = s * kStep + e * 32 + g4 * 8 < g.K;
                xs[e] = zero_unless(xs[e], there);
#pragma unroll
                for (int j = 0; j < RK; ++j) as[j][e] = zero_unless(as[j][e], there);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < RK; ++j) acc[j] = mfma_bf16(as[j][e], xs[e], acc[j]);
    }
    if (wave > 0)
#pragma unroll
        for (int j = 0; j < RK; ++j) lds[wave - 1][j][l] = acc[j];
    __syncthreads();
    if (wave > 0) return;
    // lane: ranks 4 g4 .. of row c
#pragma unroll
    for (int j = 0; j < RK; ++j) {
        const f32x4 v = ((acc[j] + lds[0][j][l]) + lds[1][j][l]) + lds[2][j][l];
        const int rank = j * 16 + g4 * 4;
        if (c < tl.count && rank < g.r)
            *reinterpret_cast<f32x4*>(g.part + ((size_t)split * g.M + tl.start + c) * g.r + rank) = v;
    }
}

// Prompt tiles: 64 rows, 16 a wave, x and a through a ring of D steps in LDS, filled by
// DMA. Bound by the stream of x; a tile reads its adapter's a once for 64 rows. A DMA
// moves 8 rows x 128 bytes, whole lines: in the operands' own order, 16 rows x 64 bytes,
// the L2 gave half the rate. The 16-byte pieces of a row lie in LDS XOR-ed by the row, so
// that the operands' reads have no bank conflicts.
template <int RK, int D>
__global__ __launch_bounds__(256) void shrink_ring_kernel(LoraArgs g)
{
    constexpr int PIECES = (4 + RK) * 2, PW = (PIECES + 3) / 4;       // a step's; a wave's
    __shared__ __attribute__((aligned(16))) uint8_t lds[D][PIECES * 1024];
    const PlanHeader h = *g.plan;
    int tile, split;
    tile_and_part(g.xcds, g.splits, tile, split);
    if (!plan_fits(h, g) || tile >= h.n_tiles) return;
    const Tile tl = plan_tiles(g.plan)[tile];
    if (tl.adapter < 0) return;
    const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (g.K + kStep - 1) / kStep;
    const int s0 = (int)((long)steps * split / g.splits), s1 = (int)((long)steps * (split + 1) / g.splits);
    const int* rows = plan_rows(g.plan, g.M, g.n_adapters) + tl.start;
    // Piece p: rows 8 p .. of x (p < 8), then ranks 8 (p - 8) .. of a. A wave's spare turn
    // repeats the last piece.
    const uint16_t* from[PW];
    int piece[PW];
    const int k_lane = ((l & 7) ^ (l >> 3)) * 8;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        piece[i] = min(wave * PW + i, PIECES - 1);
        const int r = piece[i] * 8 + (l >> 3);
        from[i] = piece[i] < 8 ? g.x + (size_t)rows[min(r, tl.count - 1)] * g.K
                               : g.a + ((size_t)tl.adapter * g.r + min(r - 64, g.r - 1)) * g.K;
    }
    auto fetch = [&](int s) {
        // (a piece past K: the row's end again, dropped below)
        const int k = min(s * kStep + k_lane, g.K - 8);
#pragma unroll
        for (int i = 0; i < PW; ++i)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(from[i] + k),
                (__attribute__((address_space(3))) void*)(lds[(s - s0) % D] + piece[i] * 1024), 16, 0, 0);
    };
    f32x4 acc[RK];
#pragma unroll
    for (int j = 0; j < RK; ++j) acc[j] = f32x4{0, 0, 0, 0};
    wait_vm<0>();               // (nothing but steps on its way below)
    for (int s = s0; s < min(s0 + D - 1, s1); ++s) fetch(s);
    // the lane's row c, K pieces g4 and 4 + g4 of the step
    const int at[2] = {c * 128 + (g4 ^ (c & 7)) * 16, c * 128 + ((4 + g4) ^ (c & 7)) * 16};
    for (int s = s0; s < s1; ++s) {
        wait_steps<PW, D - 2>(min(D - 2, s1 - 1 - s));
        stage_barrier();        // the step is there, and nobody reads the one before it
        if (s + D - 1 < s1) fetch(s + D - 1);
        const uint8_t* base = lds[(s - s0) % D];
        bf16x8 x[2], a[RK][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            x[e] = *reinterpret_cast<const bf16x8*>(base + wave * 2048 + at[e]);
#pragma unroll
            for (int j = 0; j < RK; ++j)
                a[j][e] = *reinterpret_cast<const bf16x8*>(base + (4 + j) * 2048 + at[e]);
        }
        if (s * kStep + kStep > g.K)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool there = s * kStep + e * 32 + g4 * 8 < g.K;
                x[e] = zero_unless(x[e], there);
#pragma unroll
                for (int j = 0; j < RK; ++j) a[j][e] = zero_unless(a[j][e], there);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < RK; ++j) acc[j] = mfma_bf16(a[j][e], x[e], acc[j]);
    }
    const int row = wave * 16 + c;
#pragma unroll
    for (int j = 0; j < RK; ++j) {
        const int rank = j * 16 + g4 * 4;
        if (row < tl.count && rank < g.r)
            *reinterpret_cast<f32x4*>(g.part + ((size_t)split * g.M + tl.start + row) * g.r + rank) = acc[j];
    }
}

// The values of lanes 0..31 (j = 0) or 32..63 (j = 1) in both halves of the wave.
__device__ __forceinline__ bf16x8 half_of(const bf16x8& x, int j)
{
    i32x4 w = __builtin_bit_cast(i32x4, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap((unsigned)w[i], (unsigned)w[i], false, false);
        w[i] = (int)r[j];
    }
    return __builtin_bit_cast(bf16x8, w);
}

// F operand pieces of 32 ranks (F = 0: 16 ranks, the remainders in the other half of
// one piece). Outputs transposed, b as the first operand with its rows in the order that
// leaves eight consecutive columns of a row in a lane. A wave takes U steps of 32 columns
// at a time, all their loads of base and b at once, the first ones before t is joined.
// Bound by these streams.
template <int RT, int F, bool F32, int U>
__global__ __launch_bounds__(256) void expand_kernel(LoraArgs g)
{
    constexpr int P = F == 0 ? 1 : F, PARTS = F == 0 ? 1 : 2, BW = F32 ? 2 : 1;
    __shared__ bf16x8 lds[RT][P][PARTS][64];
    const PlanHeader h = *g.plan;
    const int chunks = (g.N + g.n_chunk - 1) / g.n_chunk;
    int tile, n0;
    tile_and_part(g.xcds, chunks, tile, n0);
    n0 *= g.n_chunk;
    if (!plan_fits(h, g) || tile >= h.n_tiles) return;
    const Tile tl = plan_tiles(g.plan)[tile];
    const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_end = min(n0 + g.n_chunk, g.N);
    const int* rows = plan_rows(g.plan, g.M, g.n_adapters) + tl.start;
    if (tl.adapter < 0) {                       // no adapter: c = base
        if (g.c == g.base) return;
        constexpr int E = F32 ? 4 : 8, B = 4;
        const int per = (n_end - n0) / E, all = per * tl.count;
        for (int v = threadIdx.x; v < all; v += 256 * B) {
            i32x4 w[B];
            size_t at[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int e = min(v + i * 256, all - 1);
                at[i] = ((size_t)rows[e / per] * g.N + n0 + e % per * E) * (F32 ? 4 : 2);
                w[i] = ldg16(static_cast<const uint8_t*>(g.base) + at[i]);
            }
#pragma unroll
            for (int i = 0; i < B; ++i)
                *reinterpret_cast<i32x4*>(static_cast<uint8_t*>(g.c) + at[i]) = w[i];
        }
        return;
    }
    int row[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) row[i] = rows[min(i * 16 + c, tl.count - 1)];
    const uint16_t* b = g.b + (size_t)tl.adapter * g.N * g.r;
    // Past the chunk's end the last columns again, past the tile's its last row: what is
    // not stored.
    const int rank0 = F == 0 ? (g4 & 1) * 8 : g4 * 8;
    i32x4 base[U][RT][BW];
    // (16 ranks: one load brings both halves of the columns, j = lane / 32)
    constexpr int BJ = F == 0 ? 1 : 2;
    bf16x8 bs[U][BJ][P];
    auto load = [&](int n) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = n + u * 32;
#pragma unroll
            for (int j = 0; j < BJ; ++j) {
                const int bn = min(at + (c >> 2) * 8 + (F == 0 ? g4 >> 1 : j) * 4 + (c & 3), n_end - 1);
#pragma unroll
                for (int f = 0; f < P; ++f)
                    bs[u][j][f] = load8(b + (size_t)bn * g.r + min(f * 32 + rank0, g.r - 8));
            }
            const int col = min(at + g4 * 8, n_end - 8);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int e = 0; e < BW; ++e)
                    base[u][i][e] = ldg16(static_cast<const uint8_t*>(g.base) +
                                          ((size_t)row[i] * g.N + col) * (F32 ? 4 : 2) + e * 16);
        }
    };
    int n = n0 + wave * (U * 32);
    load(n);

    // t = scale * the sum of K's parts, in the operands' lane order.
    const float scale = g.scale[tl.adapter];
    const size_t split = (size_t)g.M * g.r;
    constexpr int ITEMS = (RT * P * 64 + 255) / 256;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
        const int u = threadIdx.x + it * 256;
        if (RT * P * 64 % 256 != 0 && u >= RT * P * 64) break;
        const int i = u / (P * 64), f = u / 64 % P, ul = u & 63, r = i * 16 + (ul & 15);
        const int rank = F == 0 ? (ul >> 4 & 1) * 8 : f * 32 + (ul >> 4) * 8;
        const bool there = r < tl.count && rank < g.r;
        const float* p = g.part + (size_t)(tl.start + min(r, tl.count - 1)) * g.r + min(rank, g.r - 8);
        f32x4 s[2] = {};
        auto parts = [&](auto n, int k0) {
            constexpr int NP = decltype(n)::value;
            f32x4 v[NP][2];
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                const float* q = p + (size_t)min(k0 + e, g.splits - 1) * split;
                v[e][0] = *reinterpret_cast<const f32x4*>(q);
                v[e][1] = *reinterpret_cast<const f32x4*>(q + 4);
            }
#pragma unroll
            for (int e = 0; e < NP; ++e)
                if (k0 + e < g.splits) {
                    s[0] += v[e][0];
                    s[1] += v[e][1];
                }
        };
        if (g.splits <= 4) parts(std::integral_constant<int, 4>{}, 0);
        else
            for (int k = 0; k < g.splits; k += 8) parts(std::integral_constant<int, 8>{}, k);
        bf16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = there ? s[e / 4][e % 4] * scale : 0.0f;
            hi[e] = (__bf16)v;
            // (an infinity has no remainder: inf - inf would make it NaN)
            lo[e] = (__bf16)(__builtin_isinf((float)hi[e]) ? 0.0f : v - (float)hi[e]);
        }
        if constexpr (F == 0) {
            lds[i][0][0][ul] = ul < 32 ? hi : lo;
        } else {
            lds[i][f][0][ul] = hi;
            lds[i][f][1][ul] = lo;
        }
    }
    __syncthreads();
    bf16x8 t[RT][P][PARTS];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int f = 0; f < P; ++f)
#pragma unroll
            for (int e = 0; e < PARTS; ++e) t[i][f][e] = lds[i][f][e][l];
    while (true) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = n + u * 32 + g4 * 8;        // N % 16 == 0: all eight inside or past the end
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                f32x4 v[2];
                if constexpr (F32) {
                    v[0] = __builtin_bit_cast(f32x4, base[u][i][0]);
                    v[1] = __builtin_bit_cast(f32x4, base[u][i][1]);
                } else {
                    const i32x4 x = base[u][i][0];
                    v[0] = f32x4{bf16lo(x[0]), bf16hi(x[0]), bf16lo(x[1]), bf16hi(x[1])};
                    v[1] = f32x4{bf16lo(x[2]), bf16hi(x[2]), bf16lo(x[3]), bf16hi(x[3])};
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f32x4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int f = 0; f < P; ++f) {
                        // (a rank past r: t is 0 there, and what was loaded must not be NaN)
                        bf16x8 w = zero_unless(bs[u][F == 0 ? 0 : j][f], f * 32 + rank0 < g.r);
                        if constexpr (F == 0) w = half_of(w, j);
#pragma unroll
                        for (int e = PARTS - 1; e >= 0; --e) d = mfma_bf16(w, t[i][f][e], d);
                    }
                    v[j] += d;
                }
                if (i * 16 + c < tl.count && col < n_end) {
                    const size_t o = (size_t)row[i] * g.N + col;
                    if constexpr (F32) {
                        f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(g.c) + o);
                        p[0] = v[0];
                        p[1] = v[1];
                    } else {
                        auto two = [](float x, float y) { return (uint32_t)f32_to_bf16(x) | (uint32_t)f32_to_bf16(y) << 16; };
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.c) + o) =
                            make_uint4(two(v[0][0], v[0][1]), two(v[0][2], v[0][3]),
                                       two(v[1][0], v[1][1]), two(v[1][2], v[1][3]));
                    }
                }
            }
        }
        n += U * 128;
        if (n >= n_end) break;
        load(n);
    }
}

bool sizes_ok(int M, int n_adapters)
{
    return M >= 1 && M <= (1 << 20) && n_adapters >= 1 && n_adapters <= kMaxAdapters;
}
bool rank_ok(int rank) { return rank >= 8 && rank <= 128 && rank % 8 == 0; }

// Parts of K: as many as fill the device, with few prompt tiles twice over, each at least
// a step a wave.
int k_splits(int M, int n_adapters, int K)
{
    const int steps = (K + kStep - 1) / kStep, tiles = max_tiles(M, n_adapters);
    const int want = (tile_rows(M) > 16 && tiles < 64 ? 2 : 1) * kPlanCUs / tiles;
    return std::max(1, std::min(std::min((steps + 3) / 4, want), 16));
}

void launch_shrink(const LoraArgs& g, unsigned blocks, hipStream_t s)
{
    if (g.r <= 16) shrink_kernel<1><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 32) shrink_kernel<2><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 64) shrink_kernel<4><<<blocks, 256, 0, s>>>(g);
    else shrink_kernel<8><<<blocks, 256, 0, s>>>(g);
}

void launch_shrink_ring(const LoraArgs& g, unsigned blocks, hipStream_t s)
{
    if (g.r <= 16) shrink_ring_kernel<1, 6><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 32) shrink_ring_kernel<2, 5><<<blocks, 256, 0, s>>>(g);
    else if (g.r <= 64) shrink_ring_kernel<4, 4><<<blocks, 256, 0, s>>>(g);
    else shrink_ring_kernel<8, 3><<<blocks, 256, 0, s>>>(g);
}

// Steps of 32 columns a wave loads at once (of `big` launches, whose workgroups have them
// for all four waves; 8, 4 or 6 steps for few ranks gained nothing).
template <int RT>
constexpr int expand_steps(int r)
{
    return RT == 1 || r <= 64 ? 2 : 1;
}

template <int RT, bool F32>
void launch_expand(const LoraArgs& g, bool big, unsigned blocks, hipStream_t s)
{
    auto go = [&](auto f, auto steps) {
        constexpr int F = decltype(f)::value, U = decltype(steps)::value;
        if (big) expand_kernel<RT, F, F32, U><<<blocks, 256, 0, s>>>(g);
        else expand_kernel<RT, F, F32, 1><<<blocks, 256, 0, s>>>(g);
    };
    if (g.r <= 16) go(std::integral_constant<int, 0>{}, std::integral_constant<int, expand_steps<RT>(16)>{});
    else if (g.r <= 32) go(std::integral_constant<int, 1>{}, std::integral_constant<int, expand_steps<RT>(32)>{});
    else if (g.r <= 64) go(std::integral_constant<int, 2>{}, std::integral_constant<int, expand_steps<RT>(64)>{});
    else go(std::integral_constant<int, 4>{}, std::integral_constant<int, expand_steps<RT>(128)>{});
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
    // Columns a workgroup, each of which joins the parts of t for itself: for four workgroups
    // a CU of decode tiles (two: 64 rows of 40 adapters, 2560 -> 19456, 13.6 us instead of
    // 11.4, replayed), six of a prompt's, but then 256 columns each while these fill half of the device
    // (two: 4090 rows -> 19456 111 us, 96; 128 columns: 1000 rows of rank 128 47 us, 37). A
    // wave takes its steps together where there are two rounds of them or more; the columns
    // are then whole rounds, in decode rather fewer (more: 12.3 us in the case above).
    const bool f32 = c_dtype == HEPH_DTYPE_F32, decode = tile_rows(M) == 16;
    const int round = 128 * (decode ? expand_steps<1>(rank) : expand_steps<4>(rank));
    const int least = !decode && (int64_t)tiles * (N / 256) >= kPlanCUs / 2 ? 256 : 128;
    const int chunks = std::max(1, std::min(((decode ? 4 : 6) * kPlanCUs + tiles - 1) / tiles,
                                            (N + least - 1) / least));
    const int want = (N + chunks - 1) / chunks;
    const bool big = want >= 2 * round;
    const int n_chunk = big ? (decode ? want : want + round - 1) / round * round : (want + 127) / 128 * 128;
    const int64_t expand = blocks_for(tiles, (N + n_chunk - 1) / n_chunk);
    if (expand > INT32_MAX) return HEPH_ERR_UNSUPPORTED;
    if (int st = check_device()) return st;
    const LoraArgs g{c, base, x_bf16, a_bf16, b_bf16, scale,
                     static_cast<PlanHeader*>(const_cast<void*>(plan)), static_cast<float*>(ws), M, N, K,
                     rank, n_adapters, splits, n_chunk, xcds_for(tiles)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (decode) {
        launch_shrink(g, (unsigned)blocks_for(tiles, splits), s);
        f32 ? launch_expand<1, true>(g, big, (unsigned)expand, s)
            : launch_expand<1, false>(g, big, (unsigned)expand, s);
    } else {
        launch_shrink_ring(g, (unsigned)blocks_for(tiles, splits), s);
        f32 ? launch_expand<4, true>(g, big, (unsigned)expand, s)
            : launch_expand<4, false>(g, big, (unsigned)expand, s);
    }
    return status_of(hipGetLastError());
}

}  // extern "C"
