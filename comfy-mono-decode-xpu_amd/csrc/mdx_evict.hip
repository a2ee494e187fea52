// Eviction from the paged cache by the attention weight that its tokens have drawn (mdx_page_evict; layout: mdx_pages.hip, weights:
// mdx_mass.hip).
//
// Sequence dst <- of src's n tokens, for every layer and kv head by itself, the first `sinks`, the last `recent` and, of the
// others, the `keep` with the largest mass (ties: the lowest place; NaN last), in their order; all of them if there are no more
// than that. They go to fresh pages, so shared pages stay as they are for who shares them, nothing is overwritten that
// another pair of the call reads, and src may be thinned in place or as a copy.
//
// Two launches (several of 2^20 work-groups where there are more). evict_plan_kernel: one work-group looks the sources' pages over
// and gives the fresh ones (as page_fork's plan does), the others, one per (pair, layer, kv head), find the keep-th largest mass by a
// radix search over its order-preserving bits (11 + 11 + 10, the masses in registers and LDS up to 16384 tokens, read again beyond)
// and write the kept tokens' numbers, places in the pool and masses in order. evict_move_kernel: work-groups of whole new pages
// gather the kept rows, 16 bytes a lane, and take the full pages' mean keys; the first ones change the tables.
//
// What bounds it: the kept rows' bytes, read and written (4 sequences of 16100 tokens to 2048 in 8 layers of 8 kv heads of 128: the
// move 115 us at 4.6 TB/s behind a plan of 21); for one short sequence the latency of the plan's and the search's dependent
// steps (2001 tokens to 248 in one layer: 7 us a launch).
//
// Reference: none (its cache is never thinned).
#include "mdx_pages.hpp"

namespace mdx {
namespace {

struct EvictArgs {
    unsigned char* kv;
    uint16_t* ksum;  // null: none
    int32_t* table;
    int64_t ts;
    int32_t* length;
    int32_t* refs;
    float* mass;  // [L][B][Hk][N]
    const int32_t* dst;
    const int32_t* src;
    int64_t* slots;  // [M][room] or null
    int32_t* status;
    int32_t* kept;  // [M][L][Hk][most]
    int B, W, P, T, lt, D, L, Hk, M, room, half;
    int64_t N;  // places of a row of mass
    int keep, sinks, recent, most;
    int unit, units;  // pages of a work-group of the move, and such work-groups per (pair, layer, K or V, kv head)
    // workspace
    int4* pair;      // [M]: state (1 served, 0 too few pages, -1 refused), tokens, first fresh page, the sequence stays as it is
    int32_t* fresh;  // the free pages given out
    int32_t* place;  // [M][L][Hk][most]: row page * T + t of the pool; -1: none (such a pair is refused)
    float* drawn;    // [M][L][Hk][most]
};

// ---- the plan -----------------------------------------------------------------------------------------------
__device__ void evict_plan(const EvictArgs& a) {
    __shared__ int tmp[PLAN_T / 64];
    __shared__ int sdst[MAX_SEQS], source[MAX_SEQS], pages[MAX_SEQS];
    const int i = threadIdx.x;
    const int d = i < a.M ? a.dst[i] : -1, s = i < a.M ? a.src[i] : -1;
    sdst[i] = d;
    __syncthreads();
    bool valid = i < a.M && d >= 0 && d < a.B && s >= 0 && s < a.B;
    if (valid)
        for (int j = 0; j < i; ++j) valid = valid && sdst[j] != d;  // (the first pair of a place counts)
    int n = 0, need = 0;
    bool stays = false;
    if (valid) {
        const int had = clamp_len(a.length[s], a.W, a.lt);
        stays = s == d && had <= a.most;
        n = min(had, a.most);
        const int64_t total = (int64_t(n) + a.room + a.T - 1) >> a.lt;
        if (total > a.W) {
            valid = false;
        } else if (stays) {  // only the pages of its room (and none for tokens that it has)
            valid = (n & (a.T - 1)) == 0 || uint32_t(a.table[d * a.ts + (n >> a.lt)]) < uint32_t(a.P);
            for (int j = n >> a.lt; j < int(total); ++j) need += uint32_t(a.table[d * a.ts + j]) >= uint32_t(a.P);
        } else {
            need = int(total);
        }
        source[i] = s;
        pages[i] = valid && !stays ? (had + a.T - 1) >> a.lt : 0;
    } else {
        pages[i] = 0;
    }
    // Every token that may move has to stand in a page: its new place would be attended, with what another sequence left there. The
    // pairs' entries by as many threads each.
    __syncthreads();
    int each = PLAN_T;
    while (each * a.M > PLAN_T) each >>= 1;
    const int mine = i / each;  // (a thread of no pair: its pages are 0)
    const int32_t* row = a.table + (pages[mine] ? source[mine] : 0) * a.ts;
    bool hole = false;
#pragma unroll 4
    for (int j = i % each; j < pages[mine]; j += each) hole |= uint32_t(row[j]) >= uint32_t(a.P);
    if (hole) sdst[mine] = -1;  // (a valid pair's is not)
    __syncthreads();
    valid = valid && sdst[i] >= 0;
    if (!valid) n = need = 0;
    int want = 0, upto = 0, have = 0;
    if (__syncthreads_or(need)) {
        upto = block_sum_incl(need, tmp, want);
        have = free_pages(a.refs, a.P, want, a.fresh, tmp);
    }
    const bool served = valid && (need == 0 || upto <= have);
    if (i < a.M) {
        a.pair[i] = make_int4(valid ? (served ? 1 : 0) : -1, n, upto - need, stays);
        a.status[i] = valid ? (served ? 1 : 0) : -1;
    }
}

// ---- the selection -------------------------------------------------------------------------------------------
// a mass as a number whose unsigned order is the masses' (-0 and 0 alike, NaN lowest)
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u >> 31 ? ~u : u | 0x80000000u);
}

// EACH tokens of a thread per round, side by side (of one page: those have at least 16 rows)
constexpr int BINS = 2048;

template <int EACH>
__device__ void evict_select(const EvictArgs& a, int unit) {
    constexpr int ROUND = PLAN_T * EACH;
    __shared__ int hist[BINS];
    __shared__ int tmp[PLAN_T / 64], pick[3];
    __shared__ float held[EACH][PLAN_T];  // the round's masses
    const int t = threadIdx.x, h = unit % a.Hk, l = unit / a.Hk % a.L, i = unit / (a.Hk * a.L);
    const int s = a.src[i], d = a.dst[i];
    int32_t* kept = a.kept + int64_t(unit) * a.most;
    if (s < 0 || s >= a.B) return;  // (refused: the move writes what is due)
    const float* mass = a.mass + ((int64_t(l) * a.B + s) * a.Hk + h) * a.N;
    const bool even = (reinterpret_cast<uintptr_t>(mass) & 15) == 0;
    const int places = a.W << a.lt;  // (there are as many masses: loaded ahead of the length)
    uint32_t key[EACH];
    auto load = [&](int from) {  // this thread's masses of the round
        const int t0 = from + t * EACH;
        float x[EACH];
        if (even && t0 + EACH <= places) {
#pragma unroll
            for (int j = 0; j < EACH; j += 4) {
                const float4 v = *reinterpret_cast<const float4*>(mass + t0 + j);
                x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < EACH; ++j) x[j] = t0 + j < places ? mass[t0 + j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            held[j][t] = x[j];  // (read by this thread alone)
            key[j] = order_of(x[j]);
        }
    };
    load(0);
    const int n = clamp_len(a.length[s], a.W, a.lt), first = min(a.sinks, n), last = max(first, n - a.recent);
    const int32_t* row = a.table + s * a.ts;
    int32_t* place = a.place + int64_t(unit) * a.most;
    float* drawn = a.drawn + int64_t(unit) * a.most;
    const bool all = n <= a.most;
    for (int k = (all ? n : a.most) + t; k < a.most; k += PLAN_T) kept[k] = -1;
    if (all && s == d) {  // it stays
        for (int k = t; k < n; k += PLAN_T) kept[k] = k;
        return;
    }
    // which of this thread's tokens of the round are below `end`
    auto below = [&](int from, int end) -> uint32_t {
        const int m = end - from - t * EACH;
        return m <= 0 ? 0u : m >= EACH ? (1u << EACH) - 1u : (1u << m) - 1u;
    };
    // ---- the order from which on keys are kept, and how many of the order just below it (ties)
    const bool once = n <= ROUND;
    uint32_t prefix = 0, from_key = 0;
    int left = a.keep;
    bool ties = false;
    if (!all && a.keep > 0) {
        for (int shift = 32; shift > 0;) {
            const int bits = shift == 10 ? 10 : 11, low = shift - bits;
            for (int k = t; k < BINS; k += PLAN_T) hist[k] = 0;
            __syncthreads();
            for (int from = 0; from < n; from += ROUND) {
                if (!once) load(from);
                const uint32_t in = below(from, last) & ~below(from, first);
#pragma unroll
                for (int j = 0; j < EACH; ++j)
                    if (((in >> j) & 1u) && (shift == 32 || (key[j] >> shift) == prefix)) atomicAdd(&hist[(key[j] >> low) & ((1u << bits) - 1u)], 1);
            }
            __syncthreads();
            // two bins per thread, from the top
            const int h0 = hist[BINS - 1 - 2 * t], h1 = hist[BINS - 2 - 2 * t];
            int total;
            const int before = block_sum_incl(h0 + h1, tmp, total) - h0 - h1;
            if (before < left && left <= before + h0 + h1) {
                const bool upper = left <= before + h0;
                pick[0] = BINS - 1 - 2 * t - (upper ? 0 : 1);
                pick[1] = left - before - (upper ? 0 : h0);
                pick[2] = upper ? h0 : h1;
            }
            __syncthreads();
            prefix = (prefix << bits) | uint32_t(pick[0]);
            left = pick[1];
            shift = low;
            ties = pick[2] != left;
            from_key = prefix << shift;
            if (!ties) break;  // (uniform: the whole bin is kept)
        }
    }
    // ---- the kept tokens in order
    int above = 0, equal = 0;  // kept ones and ties in the rounds before
    for (int from = 0; from < n; from += ROUND) {
        if (!once) load(from);
        const uint32_t in = below(from, n), forced = all ? in : in & (below(from, first) | ~below(from, last));
        uint32_t over = 0, same = 0;
        if (!all && a.keep > 0) {
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                over |= key[j] >= from_key ? 1u << j : 0u;
                same |= key[j] == from_key ? 1u << j : 0u;
            }
        }
        same = ties ? same & in & ~forced : 0;
        over = (over & in & ~same) | forced;
        const int up = __popc(over), at_it = __popc(same);
        int total;
        const int upto = block_sum_incl(up | (at_it << 16), tmp, total);
        int u = above + (upto & 0xFFFF) - up, e = equal + (upto >> 16) - at_it;
        above += total & 0xFFFF;
        equal += total >> 16;
        uint32_t todo = over | same;
        if (todo == 0) continue;
        const int t0 = from + t * EACH, page = row[t0 >> a.lt];
        const int base = uint32_t(page) < uint32_t(a.P) ? (page << a.lt) + (t0 & (a.T - 1)) : -1;
        while (todo) {
            const int j = __builtin_ctz(todo);
            todo &= todo - 1;
            const bool tie = (same >> j) & 1u;
            if (!tie || e < left) {
                const int k = u + min(e, left);
                kept[k] = t0 + j;
                place[k] = base < 0 ? -1 : base + j;
                drawn[k] = held[j][t];
            }
            u += tie ? 0 : 1;
            e += tie ? 1 : 0;
        }
    }
}

template <int EACH>
__global__ __launch_bounds__(PLAN_T) void evict_plan_kernel(EvictArgs a, int first) {
    if (first == 0 && blockIdx.x == 0) evict_plan(a);
    else evict_select<EACH>(a, first + int(blockIdx.x) - 1);
}

// ---- the tables and the rows --------------------------------------------------------------------------------------
__device__ void evict_tables(const EvictArgs& a, int i) {
    const int4 p = a.pair[i];
    const int t = threadIdx.x;
    int32_t* row = nullptr;
    if (p.x == 1) {
        const int d = a.dst[i], total = int((int64_t(p.y) + a.room + a.T - 1) >> a.lt);
        row = a.table + d * a.ts;
        if (p.w) {
            // (its missing entries in order: the whole row by the first wave, a ballot per 64 entries)
            int given = p.z;
            if (t < 64)
                for (int j0 = p.y >> a.lt; j0 < total; j0 += 64) {
                    const int j = j0 + t;
                    const bool miss = j < total && uint32_t(row[j]) >= uint32_t(a.P);
                    const uint64_t m = __builtin_amdgcn_ballot_w64(miss);
                    if (miss) {
                        const int e = a.fresh[given + __popcll(m & ((uint64_t(1) << t) - 1))];
                        row[j] = e;
                        a.refs[e] = 1;
                    }
                    given += __popcll(m);
                }
        } else {
            for (int j = t; j < a.W; j += 256) {
                const int old = row[j], e = j < total ? a.fresh[p.z + j] : -1;
                if (old >= 0 && old < a.P) atomicSub(a.refs + old, 1);
                if (e >= 0) a.refs[e] = 1;
                row[j] = e;
            }
        }
        if (t == 0) a.length[d] = p.y;
    } else {
        const int64_t per = int64_t(a.L) * a.Hk * a.most;
        for (int64_t k = t; k < per; k += 256) a.kept[i * per + k] = -1;
    }
    if (!a.slots) return;
    __syncthreads();  // (the row, written by other threads)
    for (int r = t; r < a.room; r += 256) {
        const int64_t at = int64_t(p.y) + r;
        const int e = row ? row[at >> a.lt] : -1;
        a.slots[int64_t(i) * a.room + r] = e >= 0 && e < a.P ? (int64_t(e) << a.lt) + (at & (a.T - 1)) : -1;
    }
}

constexpr int MOVE_BYTES = 16384;  // of a work-group of the move: whole pages of at least that
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, int first) {
    const int x = first + int(blockIdx.x) - a.M;
    if (x < 0) {
        evict_tables(a, x + a.M);
        return;
    }
    const int c = x / a.units, h = c % a.Hk, part = c / a.Hk % 2, l = c / (2 * a.Hk) % a.L, i = c / (2 * a.Hk * a.L);
    const int4 p = a.pair[i];
    const int k0 = x % a.units * a.unit << a.lt, k1 = min(p.y, k0 + (a.unit << a.lt));
    if (p.x != 1 || p.w || k0 >= k1) return;  // (uniform)
    // keys whose pages are to be summed up here are kept in LDS on their way
    __shared__ __align__(16) unsigned char rows[MOVE_BYTES];
    const bool in_lds = !part && a.ksum && (int64_t(a.unit) << a.lt) * a.D * 2 <= MOVE_BYTES;
    const int64_t list = ((int64_t(i) * a.L + l) * a.Hk + h) * a.most;
    const int32_t *place = a.place + list, *fresh = a.fresh + p.z;
    const int lanes = a.D / 8, step = 256 / lanes, sub = int(threadIdx.x) / lanes, in = int(threadIdx.x) % lanes * 16;
    const int64_t chunk = (int64_t(l) * 2 + part) * a.Hk + h;
    unsigned char* base = a.kv + ((chunk * a.P) << a.lt) * a.D * 2 + in;
    constexpr int U = 4;
    for (int k = k0 + sub; k < k1; k += U * step) {
        u32x4 v[U];
        int from[U], to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(k + u * step, k1 - 1);
            from[u] = place[at];
            to[u] = fresh[at >> a.lt];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            to[u] = (to[u] << a.lt) + ((k + u * step) & (a.T - 1));
            if (k + u * step >= k1) from[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (from[u] >= 0) v[u] = *reinterpret_cast<const u32x4*>(base + int64_t(from[u]) * a.D * 2);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (from[u] >= 0) {
                *reinterpret_cast<u32x4*>(base + int64_t(to[u]) * a.D * 2) = v[u];
                if (in_lds) *reinterpret_cast<u32x4*>(rows + (k + u * step - k0) * a.D * 2 + in) = v[u];
            }
    }
    if (part) return;
    float* mass = a.mass + ((int64_t(l) * a.B + a.dst[i]) * a.Hk + h) * a.N;
    for (int k = k0 + int(threadIdx.x); k < k1; k += 256) mass[k] = a.drawn[list + k];
    if (!a.ksum) return;
    __syncthreads();  // (the rows above, read by other waves)
    for (int j = (k0 >> a.lt) + int(threadIdx.x >> 6); j < k1 >> a.lt; j += 4) {
        const int64_t kc = int64_t(l) * a.Hk + h;
        if (in_lds) {
            const uint16_t* at = reinterpret_cast<const uint16_t*>(rows) + ((j << a.lt) - k0) * a.D;
            mean_rows(at, a.ksum + (kc * a.P + fresh[j]) * a.D, a.T, a.D, a.half, threadIdx.x & 63);
        } else {  // (a page larger than that)
            mean_key(a, kc, fresh[j], threadIdx.x & 63);
        }
    }
}

// Selections and moves of a launch: more of them take further launches. (A launch holds under 2^32 threads, and the moves go by what
// the tables could hold: 1024 pairs of 32 layers of 8 kv heads thinned to 2048 tokens are 2^24 work-groups of 256. A loop in the
// kernels cost every call registers: the move of 4 sequences of 16100 tokens 116 -> 122 us.)
constexpr int MOST_GROUPS = 1 << 20;
static_assert(MOST_GROUPS <= most_groups(PLAN_T), "");
// f(first work-group, work-groups) of every launch
template <class F>
int launches(int groups, F f) {
    for (int first = 0; first < groups; first += MOST_GROUPS) {
        f(first, dim3(unsigned(groups - first < MOST_GROUPS ? groups - first : MOST_GROUPS)));
        MDX_LAUNCHED();
    }
    return MDX_OK;
}

int64_t lists(int64_t M, int64_t L, int64_t Hk, int64_t most) { return (M * L * Hk * most + 3) / 4 * 4; }
int64_t given(int64_t M, int64_t W) { return (M * W + 3) / 4 * 4; }

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_page_evict_workspace(int64_t pairs, int64_t W, int64_t L, int64_t Hk, int64_t most) {
    if (pairs < 1 || pairs > MAX_SEQS || W < 1 || W > (int64_t(1) << 26) || L < 1 || Hk < 1 || L * Hk > 65536 || most < 1 || most > (int64_t(1) << 30) ||
        pairs * L * Hk > (int64_t(1) << 24) || pairs * L * Hk * most >= (int64_t(1) << 31))
        return 0;
    return size_t(pairs) * sizeof(int4) + size_t(given(pairs, W)) * 4 + size_t(lists(pairs, L, Hk, most)) * 8;
}

extern "C" int mdx_page_evict(void* kv, void* ksum, int32_t dtype, int64_t L, int64_t Hk, int64_t P, int64_t T, int64_t D,
                              int32_t* table, int64_t table_stride, int64_t B, int64_t W, int32_t* length, int32_t* refs,
                              float* mass, int64_t N, const int32_t* dst, const int32_t* src, int64_t pairs, int64_t keep,
                              int64_t sinks, int64_t recent, int64_t room, int64_t* slots, int32_t* status, int32_t* kept,
                              void* workspace, size_t workspace_bytes, void* stream) {
    MDX_CHECK(kv && table && length && refs && mass && dst && src && status && kept, "null pointer");
    MDX_CHECK(dtype == MDX_DT_BF16 || dtype == MDX_DT_F16, "bf16 or fp16");
    const int lt = log2_of(T);
    MDX_CHECK(lt >= 0, "page rows: a power of two in 16..1024");
    MDX_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
    MDX_CHECK(L >= 1 && Hk >= 1 && P >= 1 && L * Hk <= 65536 && (P << lt) < (int64_t(1) << 31), "layers, heads, pages (under 2^31 rows)");
    MDX_CHECK(B >= 1 && B <= (int64_t(1) << 24) && W >= 1 && (W << lt) < (int64_t(1) << 30) && table_stride >= W && table_stride <= (int64_t(1) << 26),
              "table [sequences, W], under 2^30 tokens a sequence");
    MDX_CHECK(N >= (W << lt) && N <= (int64_t(1) << 31), "mass: a place for every token that a sequence can have");
    MDX_CHECK(pairs >= 1 && pairs <= MAX_SEQS && room >= 0 && room < (int64_t(1) << 30), "1..1024 pairs, room");
    const int64_t cap = int64_t(1) << 29;
    MDX_CHECK(keep >= 0 && sinks >= 0 && recent >= 0 && keep <= cap && sinks <= cap && recent <= cap && keep + sinks + recent >= 1 &&
                  keep + sinks + recent <= (int64_t(1) << 30),
              "1..2^30 kept tokens");
    const int64_t most = keep + sinks + recent;
    MDX_CHECK(pairs * W < (int64_t(1) << 30) && pairs * L * Hk <= (int64_t(1) << 24) && pairs * L * Hk * most < (int64_t(1) << 31),
              "too many pairs times heads times kept tokens for one call");
    MDX_CHECK(aligned(kv, 16) && aligned(ksum, 16) && aligned(mass, 4), "16-byte aligned cache");
    const size_t need = mdx_page_evict_workspace(pairs, W, L, Hk, most);
    MDX_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= need, "workspace: %zu bytes, 16-byte aligned", need);
    EvictArgs a{};
    a.kv = static_cast<unsigned char*>(kv);
    a.ksum = static_cast<uint16_t*>(ksum);
    a.table = table;
    a.ts = table_stride;
    a.length = length;
    a.refs = refs;
    a.mass = mass;
    a.dst = dst;
    a.src = src;
    a.slots = slots;
    a.status = status;
    a.kept = kept;
    a.B = int(B), a.W = int(W), a.P = int(P), a.T = int(T), a.lt = lt, a.D = int(D), a.L = int(L), a.Hk = int(Hk), a.M = int(pairs), a.room = int(room);
    a.half = dtype == MDX_DT_F16;
    a.N = N;
    a.keep = int(keep), a.sinks = int(sinks), a.recent = int(recent), a.most = int(most);
    const int64_t page = T * D * 2, held = most < (W << lt) ? most : W << lt, pages = (held + T - 1) >> lt;
    a.unit = int(page >= MOVE_BYTES ? 1 : MOVE_BYTES / page);
    a.units = int((pages + a.unit - 1) / a.unit);
    a.pair = static_cast<int4*>(workspace);
    a.fresh = reinterpret_cast<int32_t*>(a.pair + pairs);
    a.place = a.fresh + given(pairs, W);
    a.drawn = reinterpret_cast<float*>(a.place + lists(pairs, L, Hk, most));
    const int64_t moves = pairs * L * 2 * Hk * a.units;  // (of at least 32 of the kept rows each, or all: under 2^28)
    MDX_CHECK(pairs + moves < (int64_t(1) << 30), "too many pairs times heads times kept tokens for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool few = (W << lt) <= 4 * PLAN_T;  // (four tokens a thread where a round of them holds a sequence)
    const int rc = launches(int(1 + pairs * L * Hk), [&](int first, dim3 groups) {
        if (few) hipLaunchKernelGGL((evict_plan_kernel<4>), groups, dim3(PLAN_T), 0, st, a, first);
        else hipLaunchKernelGGL((evict_plan_kernel<16>), groups, dim3(PLAN_T), 0, st, a, first);
    });
    if (rc != MDX_OK) return rc;
    return launches(int(pairs + moves), [&](int first, dim3 groups) { hipLaunchKernelGGL(evict_move_kernel, groups, dim3(256), 0, st, a, first); });
}
