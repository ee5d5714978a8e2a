// pages_attention.hip - attention of a batch over the paged E4M3 cache, shared
// prefixes once for their group.
//
// One pass over the keys with a running maximum and sum (a softmax's pieces over
// disjoint key sets join exactly: m = max m_i, weights 2^(m_i - m)), both
// products on v_mfma_f32_16x16x32_bf16. An E4M3 code is a bf16 value, so K and V
// enter exactly; q is bf16 already; the unnormalized probabilities are rounded
// to bf16 (at most 2^-8 relative, and the weighted mean of many of them is nearer;
// the sum takes the rounded ones too), while scores, maxima, sums and outputs stay
// f32.
//
// Scores are formed transposed, S^T = K Q^T: a lane then holds four consecutive
// keys of ONE query row in each 16-key tile, so a row's maximum and sum need two
// lane exchanges, and after exp2 the lane holds exactly the P^T operand of
// O^T = V^T P^T for the keys in the order in which V's pages store them: neither
// scores nor probabilities cross lanes, and every K and V load is 16 bytes a lane,
// 1 KB in a row.
//
// Work units: 16 to 128 query rows (tokens x the query heads of one kv head)
// times a run of pages. A group's shared pages are units of the group's rows
// together, everything else of one sequence's rows. The plan kernel lays the
// units out from the lengths in device memory; units of the same row meet in
// the workspace and merge_kernel joins them.
//
// Measured (8 kv heads, 32 heads, graph replays): 64 sequences x 4096 keys of their
// own 102 us, 5.3 TB/s of K and V; 16 prompts of 128 tokens behind 20000 keys 706 us,
// 948 TFLOP/s (a library product of 8192^3 in bf16 reaches 1240); one sequence of
// 32768 keys 24.3 us.
#include <algorithm>
#include <type_traits>

#include "pages.h"

namespace heph {
namespace {

constexpr int kMagic = 0x41505033;
constexpr int kSlots = 512;           // workgroups that run at once: two a CU
constexpr int kMaxSeqs = HEPH_PAGES_MAX_SEQS;

struct PlanHeader {
    int magic, n_tok, n_seqs, n_groups, table_pages, n_heads, n_kv, n_units;
    int merges, pad[3];            // whether any row has other than one unit
};
// Rows row0 .. row0+rows-1 (row = token * G + head of the group, from token
// tok0 on) over pages page0 .. page0+pages-1 of table row seq. part: the
// unit's number among those of its rows, counted within the prefix (prefix
// != 0) or behind the row's prefix units.
struct Unit {
    int seq, tok0, row0, rows, page0, pages, part, prefix;
};
// Per token: keys it attends to (-1: no sequence), how many prefix and own units hold
// any of them, and where its first row's partial results lie among a kv head's: those of
// unit k at prefix + k * prefix_step, own + k * own_step.
struct Token {
    int limit, n_prefix, n_own, prefix, prefix_step, own, own_step, pad;
};

// Query rows of a unit by how many there are: 16, 32 or 64 (attend_narrow: a
// wave takes 16 rows, waves left over split the pages) or as many whole tokens
// as 128 rows hold (attend_wide).
constexpr int kNarrow = 64;
__host__ __device__ __forceinline__ int wide_rows(int G) { return 128 / G * G; }

// Pages a unit has at least: fewer would not keep the four waves of a narrow one
// busy, and writing and joining a wide one's 128 rows would outweigh its pages (4 pages
// instead of 8: two prefixes of 64 pages, 32 sequences each, beside 1000 keys a sequence,
// four layers 156 us instead of 134, 16 pages 158; alone, a prefix of 48 pages for 32
// sequences gained from 4, 21.2 us -> 17.2. Narrow units of 8 pages: four sequences behind
// 512 shared keys, four layers, 45.2 us instead of 41.6).
constexpr int kMinNarrow = 4, kMinWide = 8;

struct Sizes {
    int n_tok, n_seqs, n_groups, n_heads, n_kv;
    __host__ __device__ int group() const { return n_heads / n_kv; }
    __host__ __device__ long rows() const { return (long)n_tok * n_heads; }
    // Workgroups of one kv head that run at once.
    __host__ __device__ int slots() const { return kSlots / n_kv > 0 ? kSlots / n_kv : 1; }
    // Partial results a kv head may write: every row twice (behind a prefix, and its
    // own), and the rows of the units that splitting adds.
    __host__ __device__ long max_parts() const
    {
        return 2L * n_tok * group() + 3L * slots() * wide_rows(group());
    }
    // Units a plan may hold: one a tile (each sequence's and each group's last
    // one may be short), and a round more where long runs are split and where
    // the last round's tiles are.
    __host__ __device__ long max_units() const
    {
        const long tiles = (long)n_tok * group() / wide_rows(group());
        return 2L * slots() + n_seqs + n_groups + 2 * tiles;
    }
};

__host__ __device__ inline Token* plan_tokens(PlanHeader* p) { return reinterpret_cast<Token*>(p + 1); }
__host__ __device__ inline Unit* plan_units(PlanHeader* p, int n_tok)
{
    return reinterpret_cast<Unit*>(plan_tokens(p) + n_tok);
}

// ------------------------------------------------------------------- plan ----

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }
__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((unsigned)a + (unsigned)b - 1) / (unsigned)b); }

struct PlanArgs {
    PlanHeader* plan;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* group_start;
    const int32_t* shared;
    Sizes s;
    int table_pages;
};

// The plan kernel's inputs in LDS, loaded all at once: what follows reads them
// in chains.
struct PlanLds {
    int32_t q_start[kMaxSeqs + 1], kv_len[kMaxSeqs], group_start[kMaxSeqs + 1], shared[kMaxSeqs];
    // before each sequence: how many have less than 64 rows, with 2^16 times how many have
    // 64, and the tokens of the former
    int32_t few[kMaxSeqs + 1], few_tokens[kMaxSeqs + 1];
};

// Rows that work on the same pages: a group's on its shared ones, or one
// sequence's on its own. Tiles are numbered over all sources from `base` on, a
// sequence's last (longest) tile first.
struct Source {
    int seq, tok0, n_tok, page0, pages, kv;     // kv: 0 for a group
    int tile, tiles, base;
    int chunks;                                 // a tile's units before the last round
    int parts, units;                           // where its partial results and units start
};

struct SeqTokens {
    Source x;
    int group;
};

// How the last round's tiles are cut.
struct Rounds {
    int first, chunks;
};

__device__ __forceinline__ void set_tiles(Source& x, int G)
{
    const int rows = x.n_tok * G;
    x.tile = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= kNarrow ? kNarrow : wide_rows(G);
    x.tiles = x.pages > 0 ? ceil_div(rows, x.tile) : 0;
}

// The group's sequences and shared pages; none where sharing gains nothing. Sequences of
// more than 64 rows are bound by the matrix cores and re-read a prefix from the caches; in a
// shared one each of their rows pays another partial result, 1.5 KB written and read. It is
// shared for the others, two or more, if the pages that they need not stream again, 16 KB
// each, outweigh that (not shared and shared: 64 single tokens and a prompt of 1100 behind 64
// pages 185 us, 171; 16 and 500 behind 32 pages 53, 47). Sequences of 64 rows stream too (attend_narrow), but
// pay for 64 rows each: they count where the prefix is long and what they stream of it
// again is 16 MB or more (100 own keys each; 64 of 16 tokens, 32 + 8 heads: 256 pages
// 479 us -> 288, 64 pages 135 -> 98, but 16 pages 47 -> 56; 16 of one token, 64 + 1 heads:
// 256 pages 39 -> 35; four of them 22 -> 27).
constexpr int kLongPrefix = 32;
__device__ Source group_source(const PlanLds& in, const PlanArgs& a, int g)
{
    const int s0 = clampi(in.group_start[g], 0, a.s.n_seqs);
    const int s1 = clampi(in.group_start[g + 1], s0, a.s.n_seqs);
    const int t0 = clampi(in.q_start[s0], 0, a.s.n_tok), t1 = clampi(in.q_start[s1], t0, a.s.n_tok);
    int pages = clampi(in.shared[g], 0, a.table_pages);
    const int counts = in.few[s1] - in.few[s0], full = counts >> 16;
    const bool again = pages >= kLongPrefix && (long)(full - 1) * pages * a.s.n_kv >= 1024;
    const int few = (counts & 0xFFFF) + (again ? full : 0);
    const long many_rows = (long)(t1 - t0 - (in.few_tokens[s1] - in.few_tokens[s0])) * a.s.group();
    if (few < 2 || many_rows > 10L * (few - 1) * pages) pages = 0;
    Source x{s0, t0, t1 - t0, 0, pages, 0};
    set_tiles(x, a.s.group());
    return x;
}

__device__ Source seq_source(const PlanLds& in, const PlanArgs& a, int s, int& group)
{
    const int t0 = clampi(in.q_start[s], 0, a.s.n_tok), t1 = clampi(in.q_start[s + 1], t0, a.s.n_tok);
    const int kv = clampi(in.kv_len[s], 0, a.table_pages * kPage);
    int lo = 0, hi = a.s.n_groups;            // the last group that starts at s or before
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (in.group_start[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    group = lo > 0 && s < in.group_start[lo] ? lo - 1 : -1;
    const int page0 = group >= 0 ? group_source(in, a, group).pages : 0;
    Source x{s, t0, t1 - t0, page0, max((kv + kPage - 1) / kPage - page0, 0), kv};
    set_tiles(x, a.s.group());
    return x;
}

// Keys that token i of the source attends to.
__device__ __forceinline__ int limit_of(const Source& x, int i) { return max(x.kv - x.n_tok + i + 1, 0); }

// Tiles of the source that belong to the last round: those numbered last, r < the result.
__device__ __forceinline__ int last_round(const Source& x, const Rounds& rounds)
{
    return x.tile > kNarrow ? clampi(x.base + x.tiles - rounds.first, 0, x.tiles) : 0;
}

// Units of tile r and pages of each: a sequence's tile sees its last token's keys.
struct Cut {
    int per, chunks;
};
__device__ __forceinline__ Cut cut_tile(const Source& x, const Rounds& rounds, int G, int r)
{
    int pages = x.pages;
    if (x.kv > 0 && x.tiles > 1) {
        const int last = (int)min((unsigned)((r + 1) * x.tile) / (unsigned)G, (unsigned)x.n_tok) - 1;
        pages = clampi((limit_of(x, last) + kPage - 1) / kPage - x.page0, 0, pages);
    }
    Cut c;
    c.chunks = r < last_round(x, rounds) ? rounds.chunks : x.chunks;
    c.per = max(ceil_div(pages, c.chunks), 1);
    return c;
}

// Partial results of the tiles before r, which are full ones: one a row and unit.
__device__ __forceinline__ int parts_before(const Source& x, const Rounds& rounds, int r)
{
    const int last = last_round(x, rounds);
    return x.tile * (min(r, last) * rounds.chunks + max(r - last, 0) * x.chunks);
}

// Units of c that hold any of the first `keys` keys.
__device__ __forceinline__ int parts_seen(int keys, const Cut& c)
{
    return keys <= 0 ? 0 : min(c.chunks, ceil_div((keys + kPage - 1) / kPage, c.per));
}

// Inclusive prefix sum over the wave: within rows of 16 lanes by shifts, then each row's
// total to the rows behind it.
__device__ __forceinline__ int wave_scan(int v)
{
    auto add = [&](auto ctrl, auto rows) {
        v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});      // row_bcast 15
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});      // row_bcast 31
    return v;
}

// Exclusive prefix sums over the workgroup of the groups' values and, behind them all, the
// sequences'; the total.
__device__ int scan_block(int& g, int& s, int2* red)
{
    const int t = threadIdx.x, l = t & 63, waves = blockDim.x / 64;
    const int x = wave_scan(g), y = wave_scan(s);
    __syncthreads();
    if (l == 63) red[t / 64] = make_int2(x, y);
    __syncthreads();
    int before_g = 0, before_s = 0, all_g = 0, all_s = 0;
    for (int i = 0; i < waves; ++i) {
        const int2 r = red[i];
        if (i < t / 64) {
            before_g += r.x;
            before_s += r.y;
        }
        all_g += r.x;
        all_s += r.y;
    }
    g = before_g + x - g;
    s = all_g + before_s + y - s;
    return all_g + all_s;
}

// One thread a sequence and a group. Every workgroup repeats that and writes a share
// of the tokens; the first one also writes the units and the header.
constexpr int kPlanTokens = 64;
__global__ __launch_bounds__(kMaxSeqs) void plan_kernel(PlanArgs a)
{
    __shared__ PlanLds in;
    __shared__ Source groups[kMaxSeqs];
    __shared__ SeqTokens seqs[kMaxSeqs];
    __shared__ float2 red_f[kMaxSeqs / 64];
    __shared__ int2 red_i[kMaxSeqs / 64];
    __shared__ int merges;
    const int t = threadIdx.x, G = a.s.group(), nt = blockDim.x;
    constexpr int cap = 64;                    // (merge_row takes two lanes' worth)
    Token* tokens = plan_tokens(a.plan);
    Unit* units = plan_units(a.plan, a.s.n_tok);
    {
        // (all loads at once; the threads behind the last sequence or group repeat its entry)
        const int s = min(t, a.s.n_seqs - 1), g = min(t, a.s.n_groups - 1);
        const int start = a.q_start[s], end = a.q_start[a.s.n_seqs], kv = a.kv_len[s];
        int group_start = 0, group_end = 0, shared = 0;
        if (a.s.n_groups) {
            group_start = a.group_start[g];
            group_end = a.group_start[a.s.n_groups];
            shared = a.shared[g];
        }
        in.q_start[s] = start;
        in.kv_len[s] = kv;
        if (a.s.n_groups) {
            in.group_start[g] = group_start;
            in.shared[g] = shared;
        }
        if (t == 0) {
            in.q_start[a.s.n_seqs] = end;
            in.group_start[a.s.n_groups] = group_end;
        }
    }
    if (t == 0) merges = 0;
    __syncthreads();
    {
        int n = 0, mine = 0;
        if (t < a.s.n_seqs) {
            const int t0 = clampi(in.q_start[t], 0, a.s.n_tok);
            n = clampi(in.q_start[t + 1], t0, a.s.n_tok) - t0;
            mine = n * G == kNarrow ? 1 << 16 : n > 0 && n * G < kNarrow;
            if (n * G >= kNarrow) n = 0;
        }
        int few = mine, few_tokens = n;
        scan_block(few, few_tokens, red_i);         // (few_tokens: behind few's total, in all of them)
        if (t == 0) {
            in.few[0] = few;
            in.few_tokens[0] = few_tokens;
        }
        if (t < a.s.n_seqs) {
            in.few[t + 1] = few + mine;
            in.few_tokens[t + 1] = few_tokens + n;
        }
        __syncthreads();
    }
    Source xg{}, xs{};
    int group = -1;
    if (t < a.s.n_groups) xg = group_source(in, a, t);
    if (t < a.s.n_seqs) xs = seq_source(in, a, t, group);

    // Work: a page of a narrow unit costs the stream of its 16 KB, one of a wide unit
    // about twice that in matrix work. (In f32: it only sets a split.)
    auto wide = [](const Source& x) { return x.tile > kNarrow; };
    auto pages = [&](const Source& x, bool w) { return wide(x) == w ? (float)x.tiles * (float)x.pages : 0.0f; };
    float work_n = pages(xg, false) + pages(xs, false), work_w = pages(xg, true) + pages(xs, true);
    for (int o = 32; o; o >>= 1) {
        work_n += __shfl_xor(work_n, o);
        work_w += __shfl_xor(work_w, o);
    }
    if ((t & 63) == 0) red_f[t / 64] = make_float2(work_n, work_w);
    xg.base = wide(xg) ? xg.tiles : 0;
    xs.base = wide(xs) ? xs.tiles : 0;
    const int wide_tiles = scan_block(xg.base, xs.base, red_i);
    work_n = work_w = 0.0f;
    for (int i = 0; i < nt / 64; ++i) {
        work_n += red_f[i].x;
        work_w += red_f[i].y;
    }

    // Narrow runs are split so that the units fill the slots of a kv head, into `cap` units
    // at most (262144 keys of one sequence, 4 heads a kv head: with one kv head, 64 of 512
    // slots, 28 us; with two, 64 of 256, 32; with eight, all 64, 107). Wide tiles get
    // their share of the slots, of half of them where narrow units are a good part of the
    // work: a CU then streams for one while it multiplies for the other. Wide tiles that
    // fill the slots by themselves stay whole, but for those of a last round that would
    // leave half of the slots or more empty.
    const int slots = a.s.slots(), rest = wide_tiles % slots;
    const float tau = fmaxf((work_n + 2.0f * work_w) / (float)slots, (float)kMinNarrow);
    const float share = (float)(work_n > 0.5f * work_w ? (slots + 1) / 2 : slots) / fmaxf(work_w, 1.0f);
    auto chunks = [&](const Source& x) {
        if (!wide(x)) return clampi((int)ceilf((float)x.pages / tau), 1, cap);
        if (wide_tiles >= slots) return 1;
        return clampi(min((int)((float)x.pages * share), x.pages / kMinWide), 1, cap);
    };
    Rounds rounds{INT32_MAX, 1};
    if (wide_tiles >= slots && rest > 0)
        rounds = Rounds{wide_tiles - rest, min(min(slots / rest, cap), ceil_div(a.table_pages, kMinNarrow))};
    xg.chunks = chunks(xg);
    xs.chunks = chunks(xs);
    auto count = [&](const Source& x) {
        const int last = last_round(x, rounds);
        return (x.tiles - last) * x.chunks + last * rounds.chunks;
    };
    auto rows_in = [&](const Source& x, int r) { return min(x.tile, x.n_tok * G - r * x.tile); };
    auto parts = [&](const Source& x) {
        if (x.tiles == 0) return 0;
        const int r = x.tiles - 1;
        return parts_before(x, rounds, r) + rows_in(x, r) * cut_tile(x, rounds, G, r).chunks;
    };
    xg.parts = parts(xg);
    xs.parts = parts(xs);
    scan_block(xg.parts, xs.parts, red_i);
    xg.units = count(xg);
    xs.units = count(xs);
    // a row of another number of units than one: behind a prefix, in a split run, without keys
    if (xg.tiles > 0 || (xs.n_tok > 0 && (xs.kv < xs.n_tok || xs.tiles == 0 || xs.units > xs.tiles)))
        merges = 1;
    const int all_units = scan_block(xg.units, xs.units, red_i);
    const int max_units = (int)min(a.s.max_units(), (long)INT32_MAX);
    if (t < a.s.n_groups) groups[t] = xg;
    if (t < a.s.n_seqs) seqs[t] = SeqTokens{xs, group};
    __syncthreads();
    const int n_units = min(all_units, max_units);
    if (blockIdx.x == 0 && t == 0)
        *a.plan = PlanHeader{kMagic, a.s.n_tok, a.s.n_seqs, a.s.n_groups, a.table_pages, a.s.n_heads,
                             a.s.n_kv, n_units, merges, {}};
    // Units: a source's tiles from its last on, each one's runs in order.
    for (int u = blockIdx.x * nt + t; u < n_units; u += gridDim.x * nt) {
        auto source = [&](int i) -> const Source& {
            return i < a.s.n_groups ? groups[i] : seqs[i - a.s.n_groups].x;
        };
        int lo = 0, hi = a.s.n_groups + a.s.n_seqs;   // the last source that starts at u or before
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (source(mid).units <= u) lo = mid + 1;
            else hi = mid;
        }
        const Source x = source(max(lo - 1, 0));
        const int at = u - x.units, last = last_round(x, rounds), whole = (x.tiles - last) * x.chunks;
        // (none of the source's where the counts wrapped: q_start falls)
        Unit unit{0, 0, 0, 0, 0, 0, 0, 0};
        if ((unsigned)at < (unsigned)count(x)) {
            const int in_last = max(at - whole, 0), k = at < whole ? at % x.chunks : in_last % rounds.chunks;
            const int r = at < whole ? x.tiles - 1 - at / x.chunks : last - 1 - in_last / rounds.chunks;
            const int per = cut_tile(x, rounds, G, r).per;
            unit = Unit{x.seq, x.tok0, r * x.tile, rows_in(x, r), x.page0 + k * per,
                        min(per, x.pages - k * per), k, lo <= a.s.n_groups};
        }
        units[u] = unit;
    }
    for (int i = blockIdx.x * kPlanTokens + t; i < min(a.s.n_tok, ((int)blockIdx.x + 1) * kPlanTokens); i += nt) {
        int lo = 0, hi = a.s.n_seqs;              // the last sequence that starts at i or before
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (in.q_start[mid] <= i) lo = mid + 1;
            else hi = mid;
        }
        Token tk{-1, 0, 0, 0, 0, 0, 0, 0};
        if (lo > 0 && i < in.q_start[lo]) {
            const Source& x = seqs[lo - 1].x;
            const int g = seqs[lo - 1].group;
            tk.limit = limit_of(x, i - x.tok0);
            // units of the row's tile that hold any of `keys` keys, and where their results lie
            auto look = [&](const Source& y, int keys, int& n, int& at, int& step) {
                if (y.tiles == 0) return;
                const int row = (i - y.tok0) * G, r = (unsigned)row / (unsigned)y.tile;
                n = parts_seen(keys, cut_tile(y, rounds, G, r));
                at = y.parts + parts_before(y, rounds, r) + row - r * y.tile;
                step = rows_in(y, r);
            };
            look(x, tk.limit - x.page0 * kPage, tk.n_own, tk.own, tk.own_step);
            if (g >= 0) look(groups[g], min(tk.limit, x.page0 * kPage), tk.n_prefix, tk.prefix, tk.prefix_step);
        }
        tokens[i] = tk;
    }
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
    float* part_o;          // [n_kv][max_parts][128], unnormalized
    float2* part_ml;        // [n_kv][max_parts]: maximum (log2), sum
    Sizes s;
    int n_pages, table_pages;
};

__device__ __forceinline__ bool plan_fits(const PlanHeader& h, const AttnArgs& a)
{
    // (no branches: they would load it piece by piece)
    return ((h.magic ^ kMagic) | (h.n_tok ^ a.s.n_tok) | (h.n_seqs ^ a.s.n_seqs) |
            (h.n_groups ^ a.s.n_groups) | (h.table_pages ^ a.table_pages) |
            (h.n_heads ^ a.s.n_heads) | (h.n_kv ^ a.s.n_kv)) == 0;
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

// Max over the four lanes l, l^16, l^32, l^48, in each of them.
__device__ __forceinline__ float rows4_max(float v)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Takes the NaN codes (0x7F, 0xFF) out of 16 codes, 0 in their place; whether there were any.
__device__ __forceinline__ bool clear_nan(i32x4& w)
{
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t n = (((uint32_t)w[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
        w[i] &= (int)~(n | (n - (n >> 7)));
        any |= n;
    }
    return any != 0;
}

// exp2(x - m) of a maximum that may be -inf (nothing seen): 0, not NaN.
__device__ __forceinline__ float weight(float x, float m)
{
    return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.0f : m));
}

// Bit 4 d + i of hit[r]: this lane's row of tile r sees a NaN in V at dim 16 d + 4
// (lane / 16) + i of the page whose codes this lane reads at vp: the product of the NaN
// codes with the seen keys, both as 0 and 1. A rare path: V is read again.
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
                    const uint32_t b = (uint32_t)w[2 * h + i / 4] >> (i % 4 * 8) & 0x7Fu;
                    is_nan[i] = (__bf16)(b == 0x7F ? 1.0f : 0.0f);
                    seen[i] = (__bf16)(key0 + h * 32 + i / 4 * 16 + i % 4 < limit[r] ? 1.0f : 0.0f);
                }
                n = mfma_bf16(is_nan, seen, n);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) hit[r] |= n[i] > 0.0f ? 1u << (4 * d + i) : 0u;
        }
    }
}

// One wave's query rows: RT tiles of 16, column c of each in lane c, c+16, c+32, c+48.
template <int RT>
struct Rows {
    int tok[RT], hd[RT], limit[RT];
    int lo, hi;              // wave-uniform: smallest and largest limit of the rows
    bf16x8 q[RT][4];
    f32x4 o[8][RT];
    float m[RT];
    f32x4 sum[RT];           // four times the same value

    __device__ __forceinline__ void init(const AttnArgs& a, const Unit& u, int head, int wave_rows)
    {
        const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4, G = a.s.group();
        const Token* tokens = plan_tokens(a.plan);
        lo = INT32_MAX;
        hi = 0;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = wave_rows + r * 16 + c;
            const bool live = row < u.rows;
            const int at = u.row0 + (live ? row : 0);
            tok[r] = live ? u.tok0 + at / G : -1;
            hd[r] = head * G + at % G;
            const int keys = tokens[u.tok0 + at / G].limit;    // (no branch: all loads at once)
            limit[r] = keys & (live ? -1 : 0);
            lo = min(lo, keys | (live ? 0 : INT32_MAX));
            hi = max(hi, limit[r]);
            const uint16_t* p = a.q + (size_t)(live ? tok[r] : u.tok0) * a.q_stride + (size_t)hd[r] * kHeadDim;
#pragma unroll
            for (int f = 0; f < 4; ++f)
                q[r][f] = __builtin_bit_cast(bf16x8, ldg16(p + f / 2 * 64 + g4 * 16 + f % 2 * 8));
            m[r] = -INFINITY;
            sum[r] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d][r] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int o_ = 1; o_ < 16; o_ <<= 1) {
            lo = min(lo, __shfl_xor(lo, o_));
            hi = max(hi, __shfl_xor(hi, o_));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
    }

    // The keys of one page. k(i, h) and v(i, h) give this lane's operands from the
    // i-th 1 KB of the page's K (half i/4, keys 16 (i%4) ..; dims 8 h .. of the
    // lane's 16) and V (dims 16 i ..; the lane's keys of the page's half h). page: its
    // number in the sequence. Where some row does not see all of it, clear() takes the
    // NaN out of what v gives and says whether there was any: a NaN must reach the rows
    // that see its key and no other, and 0 * NaN is NaN; vp reads V's codes again for
    // them. AHEAD: operands come from LDS, four of them a step ahead of their products.
    template <bool AHEAD, class K, class V, class C>
    __device__ __forceinline__ void page(int page, float sc, K k, V v, C clear, const uint8_t* vp)
    {
        const int g4 = (threadIdx.x & 63) >> 4;
        f32x4 s[4][RT];
        bf16x8 w0[4], w1[4];
        auto k4 = [&](bf16x8 (&w)[4], int kt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = k(i / 2 * 4 + kt, i % 2);
        };
        auto v4 = [&](bf16x8 (&w)[4], int g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = v(2 * g + i / 2, i % 2);
        };
        auto scores4 = [&](const bf16x8 (&w)[4], int kt) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const f32x4 zero = {0, 0, 0, 0};
                    s[kt][r] = mfma_bf16(w[i], q[r][i], i ? s[kt][r] : zero);
                }
        };
        // Keeps what is on its two sides apart, so that reads stay a step ahead.
        auto step = [] { if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0); };
        if constexpr (AHEAD) {
            k4(w0, 0);
            step();
            k4(w1, 1);
            step();
            scores4(w0, 0);
            step();
            k4(w0, 2);
            step();
            scores4(w1, 1);
            step();
            k4(w1, 3);
            step();
            scores4(w0, 2);
            step();
            v4(w0, 0);
            step();
            scores4(w1, 3);
            step();
        } else {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                k4(w0, kt);
                scores4(w0, kt);
            }
        }
        if ((page + 1) * kPage > lo) {
            const int key0 = page * kPage + g4 * 4;
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + kt * 16 + i >= limit[r]) s[kt][r][i] = -INFINITY;
            if (clear()) {
                uint32_t hit[RT];
                nan_seen<RT>(vp, key0, limit, hit);
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (hit[r] >> (4 * d + i) & 1) o[d][r][i] = NAN;
            }
        }
        float top[RT];
        bool moves = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float x = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) x = fmaxf(x, s[kt][r][i]);
            // sc > 0: the largest score has the largest scaled one
            top[r] = rows4_max(x * sc);
            moves |= top[r] > m[r] + 8.0f;
        }
        // The maximum moves only by 2^8 or more: probabilities stay below 2^8, sums
        // far from f32's range, and most pages scale nothing.
        if (__any(moves)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float now = fmaxf(m[r], top[r]), f = weight(m[r], now);
                m[r] = now;
                sum[r] *= f;
#pragma unroll
                for (int d = 0; d < 8; ++d) o[d][r] *= f;
            }
        }
        bf16x8 prob[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float base = m[r] == -INFINITY ? 0.0f : m[r];
            union {
                bf16x2 p[8];
                bf16x8 v[2];
            } w;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r][i], sc, -base));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r][i + 1], sc, -base));
                    w.p[kt * 2 + i / 2] = __builtin_convertvector((f32x2){e0, e1}, bf16x2);
                }
            prob[r][0] = w.v[0];
            prob[r][1] = w.v[1];
        }
        auto add4 = [&](const bf16x8 (&w)[4], int g) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    o[2 * g + i / 2][r] = mfma_bf16(w[i], prob[r][i % 2], o[2 * g + i / 2][r]);
        };
        step();
        if constexpr (AHEAD) v4(w1, 1);
        step();
        // The sum of the rounded probabilities, as the product with a row of ones: it
        // takes what the numerators take, and the matrix cores have the time.
        const bf16x8 one = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < RT; ++r) sum[r] = mfma_bf16(one, prob[r][h], sum[r]);
        if constexpr (AHEAD) {
            add4(w0, 0);
            step();
            v4(w0, 2);
            step();
            add4(w1, 1);
            step();
            v4(w1, 3);
            step();
            add4(w0, 2);
            step();
            add4(w1, 3);
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                v4(w0, g);
                add4(w0, g);
            }
        }
    }

    // The rows' results over dim tiles d0 .. d0+nd-1, held in o[0 .. nd): to out
    // where the unit is the row's only one, else to its slot in the workspace.
    __device__ __forceinline__ void store(const AttnArgs& a, const Unit& u, int head, int d0, int nd)
    {
        const int g4 = (threadIdx.x & 63) >> 4;
        const Token* tokens = plan_tokens(a.plan);
        const float sv = a.kv_scale[a.s.n_kv + head];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (tok[r] < 0) continue;
            const Token tk = tokens[tok[r]];
            if (u.part >= (u.prefix ? tk.n_prefix : tk.n_own)) continue;    // none of its keys here
            const size_t row = (size_t)tok[r] * a.s.n_heads + hd[r];
            if (tk.n_prefix + tk.n_own == 1) {
                const float f = sum[r][0] == 0.0f && m[r] == -INFINITY ? 0.0f : sv / sum[r][0];
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
                const long part = (u.prefix ? tk.prefix + u.part * tk.prefix_step : tk.own + u.part * tk.own_step) +
                                  (hd[r] - head * a.s.group());
                // (only where a falling q_start made the plan's counts wrap)
                if ((unsigned long)part >= (unsigned long)a.s.max_parts()) continue;
                const size_t slot = (size_t)head * a.s.max_parts() + part;
                if (g4 == 0 && d0 == 0) a.part_ml[slot] = make_float2(m[r], sum[r][0]);
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    if (d < nd)
                        *reinterpret_cast<f32x4*>(a.part_o + slot * kHeadDim + (d0 + d) * 16 + g4 * 4) = o[d][r];
            }
        }
    }
};

// The ids of the 64 pages from p on, one a lane. A load among the pages' own
// would be waited for with all of them, so a run goes in blocks of 64 pages.
__device__ __forceinline__ int page_ids(const AttnArgs& a, const Unit& u, int p)
{
    const int n = p + (threadIdx.x & 63);
    return n < a.table_pages ? a.table[(size_t)u.seq * a.table_pages + n] : -1;
}

// s_waitcnt: at most N of this wave's vector memory operations and no LDS one left.
template <int N>
__device__ __forceinline__ void wait_vm()
{
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

// Up to 64 rows: a wave takes 16 of them and, where that leaves waves, every
// KW-th page of the run. Bound by the stream of K and V: the next page's 16 KB
// a wave are on their way into registers while one is worked on. (64 sequences, each
// 1024 keys 27 us, 4.9 TB/s; 64 keys 8.3 us, where a chain of four loads counts: unit,
// limits and page ids, q, pages.)
__device__ __forceinline__ void attend_narrow(const AttnArgs& a, const Unit& u, int head, int ids0, uint8_t* lds)
{
    const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4, n_kv = a.s.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KW = u.rows <= 16 ? 4 : u.rows <= 32 ? 2 : 1, kw = wave % KW;
    Rows<1> x;
    x.init(a, u, head, wave / KW * 16);
    const int end = min(u.page0 + u.pages, (x.hi + kPage - 1) / kPage);
    const float sc = a.kv_scale[head] * (0.08838834764831845f * 1.4426950408889634f);
    auto place = [&](int id) {
        // (a page that is not there is not used: any address in the pool)
        const int at = id >= 0 && id < a.n_pages ? id : 0;
        return ((size_t)at * n_kv + head) * kPageBytes + c * 64 + g4 * 16;
    };
    struct Page {
        i32x4 k[8], v[8];
        int id;
    } p0, p1;
    int ids = 0, first = 0, last = 0;
    // (past the run its last page again: a load that is left out on some path would make
    // the waits for the page before count without it, and hold up the one behind)
    auto load = [&](Page& p, int n) {
        p.id = __builtin_amdgcn_readlane(ids, min(n, last - 1) - first);
        const size_t o = place(p.id);
#pragma unroll
        for (int i = 0; i < 8; ++i) p.k[i] = ldg16(a.k_pages + o + i * 1024);
#pragma unroll
        for (int i = 0; i < 8; ++i) p.v[i] = ldg16(a.v_pages + o + i * 1024);
    };
    auto work = [&](Page& p, int n) {
        if (p.id < 0 || p.id >= a.n_pages) return;
        auto half = [](const i32x4& w, int h) { return bf16_of_codes(w[2 * h], w[2 * h + 1]); };
        auto clear = [&] {
            bool any = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) any |= clear_nan(p.v[i]);
            return __any(any);
        };
        x.page<false>(n, sc, [&](int i, int h) { return half(p.k[i], h); },
                      [&](int i, int h) { return half(p.v[i], h); }, clear,
                      a.v_pages + place(p.id));
    };
    for (first = u.page0; first < end; first += 64) {
        last = min(first + 64, end);
        ids = first == u.page0 ? ids0 : page_ids(a, u, first);
        wait_vm<0>();           // (nothing but pages on its way below)
        int n = first + kw;
        load(p0, n);
        while (n < last) {
            load(p1, n + KW);
            work(p0, n);
            n += KW;
            if (n >= last) break;
            load(p0, n + KW);
            work(p1, n);
            n += KW;
        }
    }

    // Waves on the same rows join: each takes 8 / KW of the dim tiles.
    int d0 = 0, nd = 8;
    if (KW > 1) {
        f32x4* lds_o = reinterpret_cast<f32x4*>(lds);
        float2* lds_ml = reinterpret_cast<float2*>(lds + 4 * 8 * 64 * sizeof(f32x4));
        if (g4 == 0) lds_ml[wave * 16 + c] = make_float2(x.m[0], x.sum[0][0]);
#pragma unroll
        for (int d = 0; d < 8; ++d) lds_o[(wave * 8 + d) * 64 + l] = x.o[d][0];
        __syncthreads();
        nd = 8 / KW;
        d0 = kw * nd;
        const int w0 = wave - kw;
        float top = -INFINITY, total = 0.0f;
        for (int w = 0; w < KW; ++w) top = fmaxf(top, lds_ml[(w0 + w) * 16 + c].x);
        f32x4 o[4] = {};
        for (int w = 0; w < KW; ++w) {
            const float2 ml = lds_ml[(w0 + w) * 16 + c];
            const float f = weight(ml.x, top);
            total = __builtin_fmaf(ml.y, f, total);
#pragma unroll
            for (int d = 0; d < 4; ++d)
                if (d < nd) o[d] += lds_o[((w0 + w) * 8 + d0 + d) * 64 + l] * f;
        }
        x.m[0] = top;
        x.sum[0][0] = total;
#pragma unroll
        for (int d = 0; d < 4; ++d) x.o[d][0] = o[d];
    }
    x.store(a, u, head, d0, nd);
}

// Up to 128 rows, 32 a wave. Bound by the matrix cores and the VALU's share beside
// them (exp2, maxima, conversions), so each wave converts a quarter of a page's codes
// to bf16 for all four, into one of two buffers in LDS in the operands' lane order
// (linear: free of bank conflicts), while the other is worked on; the codes of the two
// pages after that are on their way in registers (one page: 408 us instead of 371 with a
// workgroup a CU). The matrix cores are busy for half of the cycles, and the clock falls
// from 2.4 to 1.9 GHz under them: v_mfma_f32_32x32x16_bf16 with one tile's exp2 between
// the other's products took 6 % fewer cycles a page at 1.7 GHz, 745 us instead of 694.
constexpr int kWidePage = 2 * 2 * kPageBytes;      // K and V as bf16

// LDS accesses of the workgroup before and behind it are ordered; loads from
// memory stay in flight (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ void attend_wide(const AttnArgs& a, const Unit& u, int head, int ids0, uint8_t* lds)
{
    __shared__ int nan_page[2], lows[4];       // of each buffer's page; each wave's smallest limit
    const int l = threadIdx.x & 63, c = l & 15, g4 = l >> 4, n_kv = a.s.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Rows<2> x;
    x.init(a, u, head, wave * 32);
    // The run's end for all waves: a sequence's last row sees most.
    int end = u.page0 + u.pages;
    if (!u.prefix) {
        const int last = u.tok0 + (u.row0 + u.rows - 1) / a.s.group();
        end = min(end, (plan_tokens(a.plan)[last].limit + kPage - 1) / kPage);
    }
    end = __builtin_amdgcn_readfirstlane(end);
    if (l == 0) lows[wave] = x.lo;
    __syncthreads();
    // Pages that some row of any wave does not see all of: their V goes to LDS without NaN,
    // and every wave has to look for those that its rows see.
    const int lo = __builtin_amdgcn_readfirstlane(min(min(lows[0], lows[1]), min(lows[2], lows[3])));
    x.lo = lo;
    const float sc = a.kv_scale[head] * (0.08838834764831845f * 1.4426950408889634f);
    // waves 0, 1: K's 1 KB tiles 0..3, 4..7; waves 2, 3: V's
    const uint8_t* pool = (wave < 2 ? a.k_pages : a.v_pages) + (wave & 1) * 4096 + c * 64 + g4 * 16;
    for (int first = u.page0; first < end; first += 64) {
        const int last = min(first + 64, end), ids = first == u.page0 ? ids0 : page_ids(a, u, first);
        wait_vm<0>();           // (nothing but pages on its way below)
        auto id_of = [&](int n) { return __builtin_amdgcn_readlane(ids, n - first); };
        struct Codes {
            i32x4 w[4];
        } c0, c1;
        // (past the run its last page again, so that the waits count the same loads always)
        auto load = [&](Codes& x, int n) {
            const int id = id_of(min(n, last - 1)), at = id >= 0 && id < a.n_pages ? id : 0;
            const uint8_t* p = pool + ((size_t)at * n_kv + head) * kPageBytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) x.w[i] = ldg16(p + i * 1024);
        };
        auto buffer = [&](int n) { return lds + ((n - first) & 1) * kWidePage + l * 16; };
        auto convert = [&](Codes& x, int n) {
            uint8_t* to = buffer(n) + wave * 8192;
            if (wave >= 2 && (n + 1) * kPage > lo) {
                bool any = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) any |= clear_nan(x.w[i]);
                if (__any(any) && l == 0) nan_page[(n - first) & 1] = n;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<bf16x8*>(to + i * 2048) = bf16_of_codes(x.w[i][0], x.w[i][1]);
                *reinterpret_cast<bf16x8*>(to + i * 2048 + 1024) = bf16_of_codes(x.w[i][2], x.w[i][3]);
            }
        };
        // Page n, while the next one's codes (in c) go to the other buffer and the one
        // after next's are on their way: c takes the third.
        auto step = [&](Codes& codes, int n) {
            if (n + 1 < last) convert(codes, n + 1);
            load(codes, n + 3);
            const int id = id_of(n);
            if (id >= 0 && id < a.n_pages && n * kPage < x.hi) {
                const uint8_t* base = buffer(n);
                auto k = [&](int i, int h) { return *reinterpret_cast<const bf16x8*>(base + (2 * i + h) * 1024); };
                auto v = [&](int i, int h) { return k(8 + i, h); };
                auto clear = [&] { return nan_page[(n - first) & 1] == n; };
                x.page<true>(n, sc, k, v, clear,
                             a.v_pages + ((size_t)id * n_kv + head) * kPageBytes + c * 64 + g4 * 16);
            }
            lds_barrier();
        };
        load(c0, first);
        if (threadIdx.x < 2) nan_page[threadIdx.x] = -1;
        lds_barrier();          // (the last block's pages are read)
        convert(c0, first);
        load(c0, first + 1);
        load(c1, first + 2);
        lds_barrier();
        for (int n = first; n < last; n += 2) {
            step(c0, n);
            if (n + 1 >= last) break;
            step(c1, n + 1);
        }
    }
    x.store(a, u, head, 0, 8);
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_kernel(AttnArgs a)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kWidePage];
    const PlanHeader h = *a.plan;
    const int n_kv = a.s.n_kv, unit = blockIdx.x / n_kv, head = blockIdx.x % n_kv;
    // The start of a unit is a chain of loads: header, unit, then its rows' limits, q and
    // page ids together, then pages.
    const Unit u = plan_units(a.plan, a.s.n_tok)[unit];        // (the plan has room for all of the grid's)
    if (!plan_fits(h, a) || unit >= h.n_units) return;
    const int ids = page_ids(a, u, u.page0);        // (on its way while the rows are looked at)
    if (u.rows <= kNarrow) attend_narrow(a, u, head, ids, lds);
    else attend_wide(a, u, head, ids, lds);
}

// Joins the partial results of a row, two dims a lane. A row of one unit is
// finished already.
__device__ __forceinline__ void merge_row(const AttnArgs& a, const Token& tk, long row, int l)
{
    const int h = (int)(row % a.s.n_heads), n = min(tk.n_prefix + tk.n_own, 128), G = a.s.group();
    const long max_parts = a.s.max_parts();
    auto slot = [&](int k) {
        const long part = (k < tk.n_prefix ? tk.prefix + k * tk.prefix_step
                                           : tk.own + (k - tk.n_prefix) * tk.own_step) + h % G;
        return (size_t)(h / G) * max_parts + ((unsigned long)part < (unsigned long)max_parts ? part : 0);
    };
    float2 ml[2];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ml[i] = i * 64 + l < n ? a.part_ml[slot(i * 64 + l)] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[i].x);
    }
    top = wave_fold_max64(top);
    const float f0 = weight(ml[0].x, top), f1 = weight(ml[1].x, top);
    const float sum = wave_fold_sum64(__builtin_fmaf(ml[0].y, f0, ml[1].y * f1));
    const float2* part = reinterpret_cast<const float2*>(a.part_o) + l;
    float x = 0.0f, y = 0.0f;
    auto add = [&](auto parts, int k) {
        constexpr int P = decltype(parts)::value;
        float2 o[P];
#pragma unroll
        for (int i = 0; i < P; ++i) o[i] = part[slot(min(k + i, n - 1)) * (kHeadDim / 2)];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float f = __int_as_float(__builtin_amdgcn_readlane(
                __float_as_int(k + i < 64 ? f0 : f1), (k + i) & 63));
            if (k + i < n) {
                x = __builtin_fmaf(o[i].x, f, x);
                y = __builtin_fmaf(o[i].y, f, y);
            }
        }
    };
    // (as many loads on their way as there are parts, up to 16: one sequence of 32768 keys
    // 24.3 us, 25.7 with eight always; four tokens behind 512 keys, four layers, 42.0 and 42.6)
    if (n <= 4) add(std::integral_constant<int, 4>{}, 0);
    else if (n <= 8) add(std::integral_constant<int, 8>{}, 0);
    else
        for (int k = 0; k < n; k += 16) add(std::integral_constant<int, 16>{}, k);
    const float f = sum == 0.0f && top == -INFINITY ? 0.0f
                                                    : a.kv_scale[a.s.n_kv + h / a.s.group()] / sum;
    *reinterpret_cast<uint32_t*>(a.out + row * kHeadDim + 2 * l) =
        (uint32_t)f32_to_bf16(x * f) | (uint32_t)f32_to_bf16(y * f) << 16;
}

// One wave a row at a time; nothing to do where every row has one unit.
constexpr int kMergeBlocks = 2048;
__global__ __launch_bounds__(256) void merge_kernel(AttnArgs a)
{
    PlanHeader head = *a.plan;
    // each lane looks at one of the wave's next 64 rows
    const long step = (long)gridDim.x * 4, rows = a.s.rows();
    for (long row0 = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row0 < rows; row0 += 64 * step) {
        const long row = row0 + (threadIdx.x & 63) * step;
        const Token tk = plan_tokens(a.plan)[min(row, rows - 1) / a.s.n_heads];
        // (loaded beside the header, not behind its check)
        asm volatile("" : "+s"(head.magic) : "v"(tk.limit), "v"(tk.n_own), "v"(tk.own_step));
        if (!plan_fits(head, a) || !head.merges) return;
        const bool todo = row < rows && tk.limit >= 0 && tk.n_prefix + tk.n_own != 1;
        for (unsigned long long m = __ballot(todo); m; m &= m - 1) {
            const int k = __ffsll((long long)m) - 1;
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, k); };
            const Token t{of(tk.limit), of(tk.n_prefix), of(tk.n_own), of(tk.prefix), of(tk.prefix_step),
                          of(tk.own), of(tk.own_step), 0};
            merge_row(a, t, row0 + k * step, threadIdx.x & 63);
        }
    }
}

bool sizes_ok(int n_tok, int n_seqs, int n_groups, int n_heads, int n_kv)
{
    return heads_ok(n_heads, n_kv, kHeadDim) && n_tok >= 1 && n_seqs >= 1 && n_groups >= 0 &&
           n_groups <= n_seqs && n_tok <= (1 << 20) && n_seqs <= kMaxSeqs && n_heads <= 4096;
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
    return (size_t)n_kv_heads * s.max_parts() * (kHeadDim * sizeof(float) + sizeof(float2));
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
    const int threads = (n_seqs + 63) / 64 * 64;
    plan_kernel<<<(n_tok + kPlanTokens - 1) / kPlanTokens, threads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
        q_stride < (int64_t)n_heads * kHeadDim || out_bf16 == q_bf16)
        return HEPH_ERR_SHAPE;
    if (!aligned(out_bf16, 16) || !aligned(q_bf16, 16) || !aligned(k_pages, 16) ||
        !aligned(v_pages, 16) || !aligned(plan, 16) || !aligned(ws, 16) || q_stride % 8)
        return HEPH_ERR_ALIGN;
    if (plan_bytes < heph_pages_attention_plan_bytes(n_tok, n_seqs, n_groups, n_heads, n_kv_heads) ||
        ws_bytes < heph_pages_attention_ws_bytes(n_tok, n_seqs, n_groups, n_heads, n_kv_heads))
        return HEPH_ERR_WORKSPACE;
    AttnArgs a;
    a.s = Sizes{n_tok, n_seqs, n_groups, n_heads, n_kv_heads};
    // no unit has fewer pages than kMinNarrow unless it is its rows' only one
    const long tiles = (long)n_tok * a.s.group() / wide_rows(a.s.group()) * 2 + n_seqs + n_groups;
    const long blocks = std::min(a.s.max_units(), tiles * ((table_pages + kMinNarrow - 1) / kMinNarrow)) *
                        n_kv_heads;
    const long merges = std::min((a.s.rows() + 3) / 4, (long)kMergeBlocks);
    if (blocks > INT32_MAX) return HEPH_ERR_UNSUPPORTED;
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
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)n_kv_heads * a.s.max_parts() * kHeadDim);
    a.n_pages = n_pages;
    a.table_pages = table_pages;
    hipStream_t s = static_cast<hipStream_t>(stream);
    attention_kernel<<<(unsigned)blocks, 256, 0, s>>>(a);
    merge_kernel<<<(unsigned)merges, 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}

}  // extern "C"
