// pages_attention.hip - attention of a batch over the paged E4M3 cache, shared
// prefixes once for their group.
//
// One pass over the keys with a running maximum and sum (a softmax's pieces over
// disjoint key sets join exactly: m = max m_i, weights 2^(m_i - m)), both
// products on v_mfma_f32_16x16x32_bf16. An E4M3 code is a bf16 value, so K and V
// enter exactly; q is bf16 already; the unnormalized probabilities are rounded
// to bf16 (2^-9 relative on average, and the weighted mean of many of them is
// nearer), while scores, maxima, sums and outputs stay f32.
//
// Scores are formed transposed, S^T = K Q^T: a lane then holds four consecutive
// keys of ONE query row in each 16-key tile, so a row's maximum and sum need two
// lane exchanges, and after exp2 the lane holds exactly the P^T operand of
// O^T = V^T P^T for the keys in the order in which V's pages store them. Nothing
// goes through LDS, and every K and V load is 16 bytes a lane, 1 KB in a row.
//
// Work units: 16 to 128 query rows (tokens x the query heads of one kv head)
// times a run of pages. A group's shared pages are units of the group's rows
// together, everything else of one sequence's rows. The plan kernel lays the
// units out from the lengths in device memory; units of the same row meet in
// the workspace and merge_kernel joins them.
#include "pages.h"

namespace heph {
namespace {

constexpr int kMagic = 0x41505032;
constexpr int kTargetUnits = 512;     // workgroups the split of long key runs aims at: two a CU
constexpr int kPlanThreads = 1024;

struct PlanHeader {
    int magic, n_tok, n_seqs, n_groups, table_pages, n_heads, n_kv, n_units;
};
// Rows row0 .. row0+rows-1 (row = token * G + head of the group, from token
// tok0 on) over pages page0 .. page0+pages-1 of table row seq. part: the
// unit's number among those of its rows, counted within the prefix (prefix
// != 0) or behind the row's prefix units.
struct Unit {
    int seq, tok0, row0, rows, page0, pages, part, prefix;
};
// Per token: keys it attends to (-1: no sequence), and how many prefix and own
// units hold any of them.
struct Token {
    int limit, n_prefix, n_own, pad;
};

struct Sizes {
    int n_tok, n_seqs, n_groups, n_heads, n_kv;
    __host__ __device__ int group() const { return n_heads / n_kv; }
    __host__ __device__ long rows() const { return (long)n_tok * n_heads; }
    // Workspace slots a row: as many partial results as its units may write.
    __host__ __device__ int parts() const
    {
        const long p = (1L << 17) / rows();
        return (int)(p < 2 ? 2 : p > 96 ? 96 : p);
    }
    // Units a plan may hold: runs split to the target, one more for each
    // tile of each sequence and group.
    __host__ __device__ long max_units() const
    {
        const long tiles = (long)n_tok * group() / 128;
        return kTargetUnits / n_kv + 1 + n_seqs + n_groups + 2 * tiles;
    }
};

__host__ __device__ inline Token* plan_tokens(PlanHeader* p) { return reinterpret_cast<Token*>(p + 1); }
__host__ __device__ inline Unit* plan_units(PlanHeader* p, int n_tok)
{
    return reinterpret_cast<Unit*>(plan_tokens(p) + n_tok);
}

// ------------------------------------------------------------------- plan ----

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Query rows of a unit by how many there are: 16, 32, 64 or 128. Four waves
// share its pages (16 and 32 rows), pairs of waves do, or each wave takes 32
// rows over all pages.
__device__ __forceinline__ int tile_rows(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

struct Source {
    int seq, tok0, n_tok, page0, pages;
};

struct PlanArgs {
    PlanHeader* plan;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* group_start;
    const int32_t* shared;
    Sizes s;
    int table_pages;
};

// The group's sequences and shared pages; none where sharing gains nothing: a
// single sequence, or sequences that bring 64 rows or more each, whose own
// units are bound by the matrix cores and re-read a prefix from the caches.
__device__ Source group_source(const PlanArgs& a, int g)
{
    const int s0 = clampi(a.group_start[g], 0, a.s.n_seqs);
    const int s1 = clampi(a.group_start[g + 1], s0, a.s.n_seqs);
    const int t0 = clampi(a.q_start[s0], 0, a.s.n_tok), t1 = clampi(a.q_start[s1], t0, a.s.n_tok);
    const int n = s1 - s0;
    int pages = clampi(a.shared[g], 0, a.table_pages);
    if (n < 2 || (long)(t1 - t0) * a.s.group() >= 64L * n) pages = 0;
    return Source{s0, t0, pages ? t1 - t0 : 0, 0, pages};
}

__device__ Source seq_source(const PlanArgs& a, int s, int& kv)
{
    const int t0 = clampi(a.q_start[s], 0, a.s.n_tok), t1 = clampi(a.q_start[s + 1], t0, a.s.n_tok);
    kv = clampi(a.kv_len[s], 0, a.table_pages * kPage);
    int lo = 0, hi = a.s.n_groups;            // the last group that starts at s or before
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.group_start[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    int page0 = 0;
    if (lo > 0 && s < a.group_start[lo]) page0 = group_source(a, lo - 1).pages;
    return Source{s, t0, t1 - t0, page0, max((kv + kPage - 1) / kPage - page0, 0)};
}

__device__ long sum_block(long v, long* red)
{
    const int t = threadIdx.x;
    for (int o = 32; o; o >>= 1) v += __shfl_down(v, o);
    __syncthreads();
    if (t % 64 == 0) red[t / 64] = v;
    __syncthreads();
    long r = 0;
    for (int i = 0; i < kPlanThreads / 64; ++i) r += red[i];
    return r;
}

// Exclusive prefix sum over the workgroup, and the total.
__device__ int scan_block(int v, int* red, int& total)
{
    const int t = threadIdx.x, l = t & 63;
    int x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (l >= o) x += y;
    }
    __syncthreads();
    if (l == 63) red[t / 64] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        if (i < t / 64) before += red[i];
        total += red[i];
    }
    return before + x - v;
}

// How a source is cut: row tiles, and pages a unit so that a unit's time (in
// quarters of one wave's page of 16 rows: 32 rows cost twice, and with more
// rows fewer waves share the pages) is about tau.
struct Cut {
    int tile, tiles, per, chunks;
};
__device__ Cut cut_source(const Source& x, int G, long tau, int cap)
{
    Cut c;
    const int rows = x.n_tok * G;
    c.tile = tile_rows(rows);
    c.tiles = (rows + c.tile - 1) / c.tile;
    const int w = c.tile / 16;
    const long per = (tau + w - 1) / w;
    c.per = max((int)min(per, (long)max(x.pages, 1)), (x.pages + cap - 1) / cap);
    c.per = max(c.per, 1);
    c.chunks = (x.pages + c.per - 1) / c.per;
    if (c.chunks > 0) c.per = (x.pages + c.chunks - 1) / c.chunks;     // even
    if (c.chunks > 0) c.chunks = (x.pages + c.per - 1) / c.per;
    return c;
}

__device__ __forceinline__ int parts_seen(int keys, const Cut& c)
{
    return keys <= 0 ? 0 : min(c.chunks, (keys + c.per * kPage - 1) / (c.per * kPage));
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a)
{
    __shared__ long red_l[kPlanThreads / 64];
    __shared__ int red_i[kPlanThreads / 64];
    const int t = threadIdx.x, G = a.s.group(), n_src = a.s.n_groups + a.s.n_seqs;
    const int cap = a.s.parts(), cap_prefix = a.s.n_groups ? cap / 2 : 0, cap_own = cap - cap_prefix;
    const long max_units = a.s.max_units();
    Token* tokens = plan_tokens(a.plan);
    Unit* units = plan_units(a.plan, a.s.n_tok);
    // rows of no sequence
    for (int i = t; i < a.s.n_tok; i += kPlanThreads) tokens[i] = Token{-1, 0, 0, 0};
    auto source = [&](int j, int& kv) {
        kv = 0;
        return j < a.s.n_groups ? group_source(a, j) : seq_source(a, j - a.s.n_groups, kv);
    };
    long cost = 0;
    for (int j = t; j < n_src; j += kPlanThreads) {
        int kv;
        const Source x = source(j, kv);
        const int rows = x.n_tok * G, tile = tile_rows(rows);
        cost += (long)((rows + tile - 1) / tile) * x.pages * (tile / 16);
    }
    cost = sum_block(cost, red_l) * a.s.n_kv;
    const long tau = max(4L, (cost + kTargetUnits - 1) / kTargetUnits);
    int base = 0;
    for (int j0 = 0; j0 < n_src; j0 += kPlanThreads) {
        const int j = j0 + t;
        int kv = 0;
        Source x{0, 0, 0, 0, 0};
        if (j < n_src) x = source(j, kv);
        const bool prefix = j < a.s.n_groups;
        const Cut c = cut_source(x, G, tau, prefix ? cap_prefix : cap_own);
        const int n = c.tiles * c.chunks;
        int total;
        int u = base + scan_block(n, red_i, total);
        base += total;
        for (int k = 0; k < c.chunks; ++k)
            for (int r = 0; r < c.tiles; ++r, ++u)
                if (u < max_units)
                    units[u] = Unit{x.seq, x.tok0, r * c.tile, min(c.tile, x.n_tok * G - r * c.tile),
                                    x.page0 + k * c.per, min(c.per, x.pages - k * c.per), k, prefix};
        // the sequence's tokens: its own thread writes a few, the wave many
        Cut cp{16, 0, 1, 0};
        if (j < n_src && !prefix && x.page0 > 0) {
            // the group's cut, as its own thread made it
            int lo = 0, hi = a.s.n_groups;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (a.group_start[mid] <= x.seq) lo = mid + 1;
                else hi = mid;
            }
            cp = cut_source(group_source(a, lo - 1), G, tau, cap_prefix);
        }
        auto token = [&](int i, int tok0, int n_tok, int kv_, int page0, const Cut& p, const Cut& o) {
            const int limit = max(kv_ - n_tok + i + 1, 0);
            tokens[tok0 + i] = Token{limit, parts_seen(limit, p), parts_seen(limit - page0 * kPage, o), 0};
        };
        const int mine = j < n_src && !prefix ? x.n_tok : 0;
        if (mine <= 4)
            for (int i = 0; i < mine; ++i) token(i, x.tok0, x.n_tok, kv, x.page0, cp, c);
        unsigned long long many = __ballot(mine > 4);
        while (many) {
            const int l = __ffsll((long long)many) - 1;
            many &= many - 1;
            auto from = [&](int v) { return __shfl(v, l); };
            const int tok0 = from(x.tok0), nt = from(x.n_tok), kv_ = from(kv), page0 = from(x.page0);
            const Cut p{0, 0, from(cp.per), from(cp.chunks)}, o{0, 0, from(c.per), from(c.chunks)};
            for (int i = t & 63; i < nt; i += 64) token(i, tok0, nt, kv_, page0, p, o);
        }
    }
    __syncthreads();
    if (t == 0)
        *a.plan = PlanHeader{kMagic, a.s.n_tok, a.s.n_seqs, a.s.n_groups, a.table_pages, a.s.n_heads,
                             a.s.n_kv, (int)min((long)base, max_units)};
}

// -------------------------------------------------------------- attention ----

struct AttnArgs {
    uint16_t* out;
    const uint16_t* q;
    int64_t q_stride;
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    const float* kv_scale;
    const int32_t* table;
    PlanHeader* plan;
    float* part_o;          // [rows][parts][128], unnormalized
    float2* part_ml;        // [rows][parts]: maximum (log2), sum
    Sizes s;
    int n_pages, table_pages;
};

__device__ __forceinline__ bool plan_fits(const PlanHeader& h, const AttnArgs& a)
{
    return h.magic == kMagic && h.n_tok == a.s.n_tok && h.n_seqs == a.s.n_seqs &&
           h.n_groups == a.s.n_groups && h.table_pages == a.table_pages &&
           h.n_heads == a.s.n_heads && h.n_kv == a.s.n_kv;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight codes -> eight bf16 (exact).
__device__ __forceinline__ bf16x8 bf16_of_codes(int lo, int hi)
{
    union {
        bf16x2 p[4];
        bf16x8 v;
    } r;
    r.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, false);
    r.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, true);
    r.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, false);
    r.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, true);
    return r.v;
}

// Max / sum over the four lanes l, l^16, l^32, l^48, in each of them.
__device__ __forceinline__ float rows4_max(float v)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows4_sum(float v)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Bytes of w that are NaN codes (0x7F, 0xFF), as 0x80 in their place.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w)
{
    return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

// exp2(x - m) of a maximum that may be -inf (nothing seen): 0, not NaN.
__device__ __forceinline__ float weight(float x, float m)
{
    return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.0f : m));
}

// Bit 4 d + i of hit[r]: this lane's row of tile r sees a NaN code in V at dim
// 16 d + 4 (lane / 16) + i of the page at vp: the product of the NaN codes with
// the seen keys, both as 0 and 1. A rare path: V is read again, a dim tile at a time.
template <int RT>
__device__ __forceinline__ void nan_seen(const uint8_t* vp, int key0, const int (&limit)[RT],
                                         uint32_t (&hit)[RT])
{
#pragma unroll
    for (int r = 0; r < RT; ++r) hit[r] = 0;
#pragma unroll 1
    for (int d = 0; d < 8; ++d) {
        const i32x4 w = ldg16(vp + d * 1024);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            f32x4 n = {0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8 is_nan, seen;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t b = nan_bytes((uint32_t)w[2 * h + i / 4]) >> (i % 4 * 8) & 0x80u;
                    is_nan[i] = (__bf16)(b ? 1.0f : 0.0f);
                    seen[i] = (__bf16)(key0 + h * 32 + i / 4 * 16 + i % 4 < limit[r] ? 1.0f : 0.0f);
                }
                n = mfma_bf16(is_nan, seen, n);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) hit[r] |= n[i] > 0.0f ? 1u << (4 * d + i) : 0u;
        }
    }
}

// RT 16-row tiles a wave; kw of KW waves on the same rows take every KW-th page.
template <int RT>
__device__ __forceinline__ void attend(const AttnArgs& a, const Unit& u, int head, int wave_rows,
                                       int kw, int KW, f32x4* lds_o, float2* lds_ml)
{
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, c = l & 15, g4 = l >> 4;
    const int G = a.s.group(), H = a.s.n_heads, n_kv = a.s.n_kv;
    const Token* tokens = plan_tokens(a.plan);
    // this lane's rows: column c of each tile
    int tok[RT], hd[RT], limit[RT];
    int lo = INT32_MAX, hi = 0;
    bf16x8 q[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = wave_rows + r * 16 + c;
        const bool live = row < u.rows;
        const int at = u.row0 + (live ? row : 0);
        tok[r] = live ? u.tok0 + at / G : -1;
        hd[r] = head * G + at % G;
        limit[r] = live ? tokens[tok[r]].limit : 0;
        if (live) {
            lo = min(lo, limit[r]);
            hi = max(hi, limit[r]);
        }
        const uint16_t* p = a.q + (size_t)(live ? tok[r] : u.tok0) * a.q_stride + (size_t)hd[r] * kHeadDim;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const i32x4 w = ldg16(p + f / 2 * 64 + g4 * 16 + f % 2 * 8);
            q[r][f] = __builtin_bit_cast(bf16x8, w);
        }
    }
    // wave-uniform: pages below `full` need no mask, those from `end` on hold no key of ours
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int first = u.page0, end = min(u.page0 + u.pages, (hi + kPage - 1) / kPage);

    const float sc = a.kv_scale[head] * (0.08838834764831845f * 1.4426950408889634f);
    f32x4 o[8][RT];
    float m[RT], sum[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        m[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d][r] = f32x4{0, 0, 0, 0};
    }
    const int32_t* table = a.table + (size_t)u.seq * a.table_pages;
    int ids_at = first, ids = first + l < a.table_pages ? table[first + l] : -1;
    auto page_id = [&](int p) {
        if (p >= ids_at + 64) {
            ids_at = p;
            ids = p + l < a.table_pages ? table[p + l] : -1;
        }
        return __builtin_amdgcn_readlane(ids, p - ids_at);
    };
    auto page_at = [&](const uint8_t* pool, int id) {
        // (a page that is not there is not used: any address in the pool)
        const int at = id >= 0 && id < a.n_pages ? id : 0;
        return pool + ((size_t)at * n_kv + head) * kPageBytes + c * 64 + g4 * 16;
    };
    i32x4 k[8], v[8];
    int p = first + kw, id = 0;
    if (p < end) {
        id = page_id(p);
        const uint8_t* kp = page_at(a.k_pages, id);
        const uint8_t* vp = page_at(a.v_pages, id);
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = ldg16(kp + i * 1024);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ldg16(vp + i * 1024);
    }
    while (p < end) {
        const int next = p + KW;
        const bool ok = id >= 0 && id < a.n_pages;
        f32x4 s[4][RT];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
            for (int r = 0; r < RT; ++r) s[kt][r] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const i32x4 w = k[f * 4 + kt];
                const bf16x8 k0 = bf16_of_codes(w[0], w[1]), k1 = bf16_of_codes(w[2], w[3]);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    s[kt][r] = mfma_bf16(k0, q[r][2 * f], s[kt][r]);
                    s[kt][r] = mfma_bf16(k1, q[r][2 * f + 1], s[kt][r]);
                }
            }
        }
        const int id_next = next < end ? page_id(next) : -1;
        const uint8_t* vp = page_at(a.v_pages, id_next);
        if (next < end) {
            const uint8_t* kp = page_at(a.k_pages, id_next);
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = ldg16(kp + i * 1024);
        }
        if (ok) {
            const bool masked = (p + 1) * kPage > lo;
            if (masked) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p * kPage + kt * 16 + g4 * 4 + i >= limit[r]) s[kt][r][i] = -INFINITY;
                // A NaN code in V must reach the rows that see its key and no other, and
                // 0 * NaN is NaN: such codes leave V, and where a row sees one its sum is
                // set to NaN.
                uint32_t any = 0;
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) any |= nan_bytes((uint32_t)v[d][i]);
                if (__any(any != 0)) {
                    uint32_t hit[RT];
                    nan_seen<RT>(page_at(a.v_pages, id), p * kPage + g4 * 4, limit, hit);
#pragma unroll
                    for (int d = 0; d < 8; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t w = nan_bytes((uint32_t)v[d][i]);
                            v[d][i] &= (int)~(w | (w - (w >> 7)));
#pragma unroll
                            for (int r = 0; r < RT; ++r)
                                if (hit[r] >> (4 * d + i) & 1) o[d][r][i] = NAN;
                        }
                }
            }
            bf16x8 prob[RT][2];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kt][r][i]);
                // sc >= 0: the largest score has the largest scaled one
                top = rows4_max(top * sc);
                // The maximum moves only by 2^8 or more: probabilities stay below
                // 2^8, sums far from f32's range, and most pages scale nothing.
                if (__any(top > m[r] + 8.0f)) {
                    const float now = fmaxf(m[r], top), f = weight(m[r], now);
                    m[r] = now;
                    sum[r] *= f;
#pragma unroll
                    for (int d = 0; d < 8; ++d) o[d][r] *= f;
                }
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
                union {
                    bf16x2 p[8];
                    bf16x8 v[2];
                } w;
                float part = 0.0f;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r][i], sc, -base));
                        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r][i + 1], sc, -base));
                        part += e0 + e1;
                        w.p[kt * 2 + i / 2] = __builtin_convertvector((f32x2){e0, e1}, bf16x2);
                    }
                sum[r] += part;
                prob[r][0] = w.v[0];
                prob[r][1] = w.v[1];
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bf16x8 w = bf16_of_codes(v[d][2 * h], v[d][2 * h + 1]);
#pragma unroll
                    for (int r = 0; r < RT; ++r) o[d][r] = mfma_bf16(w, prob[r][h], o[d][r]);
                }
        }
        if (next < end) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = ldg16(vp + i * 1024);
        }
        p = next;
        id = id_next;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) sum[r] = rows4_sum(sum[r]);

    // Waves on the same rows join: each takes 8 / KW of the dim tiles.
    int d0 = 0, nd = 8;
    if (KW > 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (g4 == 0) lds_ml[wave * 32 + r * 16 + c] = make_float2(m[r], sum[r]);
#pragma unroll
            for (int d = 0; d < 8; ++d) lds_o[((wave * RT + r) * 8 + d) * 64 + l] = o[d][r];
        }
        __syncthreads();
        nd = 8 / KW;
        d0 = kw * nd;
        const int w0 = wave - kw;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float top = -INFINITY, total = 0.0f;
            for (int w = 0; w < KW; ++w) top = fmaxf(top, lds_ml[(w0 + w) * 32 + r * 16 + c].x);
            f32x4 x[4] = {};
            for (int w = 0; w < KW; ++w) {
                const float2 ml = lds_ml[(w0 + w) * 32 + r * 16 + c];
                const float f = weight(ml.x, top);
                total = __builtin_fmaf(ml.y, f, total);
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    if (d < nd) x[d] += lds_o[(((w0 + w) * RT + r) * 8 + d0 + d) * 64 + l] * f;
            }
            m[r] = top;
            sum[r] = total;
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d][r] = x[d];
        }
    }
    const float sv = a.kv_scale[n_kv + head];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        if (tok[r] < 0) continue;
        const Token tk = tokens[tok[r]];
        const int own_first = u.prefix ? 0 : tk.n_prefix;
        if (u.part >= (u.prefix ? tk.n_prefix : tk.n_own)) continue;       // none of its keys here
        const size_t row = (size_t)tok[r] * H + hd[r];
        if (tk.n_prefix + tk.n_own == 1) {
            const float f = sum[r] == 0.0f && m[r] == -INFINITY ? 0.0f : sv / sum[r];
            uint16_t* out = a.out + row * kHeadDim + g4 * 4;
#pragma unroll
            for (int d = 0; d < 8; ++d)
                if (d < nd) {
                    const f32x4 x = o[d][r] * f;
                    const uint2 w = make_uint2(
                        (uint32_t)f32_to_bf16(x[0]) | (uint32_t)f32_to_bf16(x[1]) << 16,
                        (uint32_t)f32_to_bf16(x[2]) | (uint32_t)f32_to_bf16(x[3]) << 16);
                    *reinterpret_cast<uint2*>(out + (d0 + d) * 16) = w;
                }
        } else {
            const size_t slot = row * a.s.parts() + own_first + u.part;
            if (g4 == 0 && d0 == 0) a.part_ml[slot] = make_float2(m[r], sum[r]);
#pragma unroll
            for (int d = 0; d < 8; ++d)
                if (d < nd)
                    *reinterpret_cast<f32x4*>(a.part_o + slot * kHeadDim + (d0 + d) * 16 + g4 * 4) = o[d][r];
        }
    }
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_kernel(AttnArgs a)
{
    __shared__ f32x4 lds_o[4 * 2 * 8 * 64];
    __shared__ float2 lds_ml[4 * 32];
    const PlanHeader h = *a.plan;
    const int n_kv = a.s.n_kv, unit = blockIdx.x / n_kv, head = blockIdx.x % n_kv;
    if (!plan_fits(h, a) || unit >= h.n_units) return;
    const Unit u = plan_units(a.plan, a.s.n_tok)[unit];
    const int wave = threadIdx.x >> 6;
    if (u.rows <= 16) {
        attend<1>(a, u, head, 0, wave, 4, lds_o, lds_ml);
    } else {
        const int KW = u.rows <= 32 ? 4 : u.rows <= 64 ? 2 : 1;
        attend<2>(a, u, head, wave / KW * 32, wave % KW, KW, lds_o, lds_ml);
    }
}

// Joins the partial results of a row: one wave a row, two dims a lane. A row of
// one unit is finished already.
__global__ __launch_bounds__(256) void merge_kernel(AttnArgs a)
{
    if (!plan_fits(*a.plan, a)) return;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.s.rows()) return;
    const int l = threadIdx.x & 63, t = (int)(row / a.s.n_heads), h = (int)(row % a.s.n_heads);
    const Token tk = plan_tokens(a.plan)[t];
    const int n = min(tk.n_prefix + tk.n_own, a.s.parts());
    if (tk.limit < 0 || n == 1) return;
    const size_t slot = (size_t)row * a.s.parts();
    float2 ml[2];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ml[i] = i * 64 + l < n ? a.part_ml[slot + i * 64 + l] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[i].x);
    }
    top = wave_fold_max64(top);
    const float f0 = weight(ml[0].x, top), f1 = weight(ml[1].x, top);
    const float sum = wave_fold_sum64(__builtin_fmaf(ml[0].y, f0, ml[1].y * f1));
    float x = 0.0f, y = 0.0f;
    for (int k = 0; k < n; ++k) {
        const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k < 64 ? f0 : f1), k & 63));
        const float2 o = *reinterpret_cast<const float2*>(a.part_o + (slot + k) * kHeadDim + 2 * l);
        x = __builtin_fmaf(o.x, f, x);
        y = __builtin_fmaf(o.y, f, y);
    }
    const float f = sum == 0.0f && top == -INFINITY ? 0.0f
                                                    : a.kv_scale[a.s.n_kv + h / a.s.group()] / sum;
    *reinterpret_cast<uint32_t*>(a.out + row * kHeadDim + 2 * l) =
        (uint32_t)f32_to_bf16(x * f) | (uint32_t)f32_to_bf16(y * f) << 16;
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
    const Sizes s{n_tok, n_seqs, n_groups, n_heads, n_kv_heads};
    return sizeof(PlanHeader) + sizeof(Token) * (size_t)n_tok + sizeof(Unit) * (size_t)s.max_units();
}

size_t heph_pages_attention_ws_bytes(int n_tok, int n_seqs, int n_groups, int n_heads,
                                     int n_kv_heads)
{
    if (!sizes_ok(n_tok, n_seqs, n_groups, n_heads, n_kv_heads)) return 0;
    const Sizes s{n_tok, n_seqs, n_groups, n_heads, n_kv_heads};
    return (size_t)s.rows() * s.parts() * (kHeadDim * sizeof(float) + sizeof(float2));
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
    const PlanArgs a{static_cast<PlanHeader*>(plan), q_start, kv_len, group_start, shared_pages,
                     Sizes{n_tok, n_seqs, n_groups, n_heads, n_kv_heads}, table_pages};
    plan_kernel<<<1, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
    AttnArgs a;
    a.s = Sizes{n_tok, n_seqs, n_groups, n_heads, n_kv_heads};
    const long blocks = a.s.max_units() * n_kv_heads, merges = (a.s.rows() + 3) / 4;
    if (blocks > INT32_MAX || merges > INT32_MAX) return HEPH_ERR_UNSUPPORTED;
    if (int st = check_device()) return st;
    a.out = static_cast<uint16_t*>(out_bf16);
    a.q = static_cast<const uint16_t*>(q_bf16);
    a.q_stride = q_stride;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.kv_scale = kv_scale;
    a.table = page_table;
    a.plan = static_cast<PlanHeader*>(const_cast<void*>(plan));
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)a.s.rows() * a.s.parts() * kHeadDim);
    a.n_pages = n_pages;
    a.table_pages = table_pages;
    hipStream_t s = static_cast<hipStream_t>(stream);
    attention_kernel<<<(unsigned)blocks, 256, 0, s>>>(a);
    merge_kernel<<<(unsigned)merges, 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
