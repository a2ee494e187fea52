// The paged cache of several sequences: sequences forked, copied, dropped (page_fork) and a step's accepted rows
// committed (page_commit), every decision on the device, so that a captured graph serves any lengths.
//
//   kv     [layers][2][Hk][P][T][D] 16-bit elements: a page of a sequence is the T rows of one page index in every
//          chunk (layer, K or V, kv head)
//   table  [B][W] page indices (-1: none); token t of sequence b is row t % T of page table[b][t / T]
//   length [B] committed tokens; refs [P] table entries that name a page (0: free)
//   ksum   [layers][Hk][P][D]: the mean key of every full page
//
// A page that holds a position at or past a sequence's length belongs to that sequence alone (page_fork copies the page
// a length ends in), so rows are written without a look at refs.
//
// Reference: none (its cache is one sequence, csrc/mtp_loop.sycl:160-196 closes accepted rows up in it; page_commit is
// that move over pages, for a batch).
#include "mdx_pages.hpp"

namespace mdx {
namespace {

constexpr int MAX_PATH = 64;      // rows of a committed path

// ---- page_fork ------------------------------------------------------------------------------------------
struct ForkArgs {
    unsigned char* kv;
    unsigned char* ksum;  // null: none
    int64_t page_bytes, sum_bytes;
    int chunks, sum_chunks;
    int32_t* table;
    int64_t ts;  // table row stride
    int32_t* length;
    int32_t* refs;
    const int32_t* dst;
    const int32_t* src;
    int64_t* slots;  // [pairs][room] or null
    int32_t* status;
    int B, W, P, T, lt, M, room, share;
    // workspace
    int32_t* head;   // [0] copies
    int32_t* pair;   // [M][4]: state (1 served, 0 too few pages, -1 refused), tokens, first fresh page, first copy
    int32_t* fresh;  // the free pages given out
    int32_t* rows;   // [M][W] new table rows
    int2* copies;    // (from, to)
};

// New table rows, the references they add, the list of copies: `nt` threads (t of them, whole waves) for pair i.
__device__ void fork_rows(const ForkArgs& a, int i, int t, int nt) {
    const int4 p = reinterpret_cast<const int4*>(a.pair)[i];
    if (p.x != 1) return;
    const int d = a.dst[i], s = a.src[i], n = p.y;
    const int full = n >> a.lt, used = (n + a.T - 1) >> a.lt, total = int((int64_t(n) + a.room + a.T - 1) >> a.lt);
    int32_t* row = a.rows + int64_t(i) * a.W;
    if (s == d) {
        // (its missing entries, -1 or otherwise no page, in order: the whole row by the first wave, a ballot per 64 entries)
        if (t >= 64) return;
        int given = p.z;
        for (int j0 = 0; j0 < a.W; j0 += 64) {
            const int j = j0 + t;
            int e = j < a.W ? a.table[d * a.ts + j] : -1;
            const bool miss = j < a.W && j >= full && j < total && uint32_t(e) >= uint32_t(a.P);
            const uint64_t m = __builtin_amdgcn_ballot_w64(miss);
            if (miss) {
                e = a.fresh[given + __popcll(m & ((uint64_t(1) << t) - 1))];
                a.refs[e] = 1;
            }
            given += __popcll(m);
            if (j < a.W) row[j] = e;
        }
        return;
    }
    const int kept = a.share ? full : 0;
    for (int j = t; j < a.W; j += nt) {
        int e = -1;
        if (j < used) e = a.table[s * a.ts + j];
        if (j < kept) {
            if (e >= 0 && e < a.P) atomicAdd(a.refs + e, 1);
            else e = -1;
        } else if (j < total) {
            const int from = e;
            e = a.fresh[p.z + j - kept];
            a.refs[e] = 1;
            if (j < used)  // (an entry that is no page leaves its copy as it was)
                a.copies[p.w + j - kept] = make_int2(from >= 0 && from < a.P ? from : -1, e);
        }
        row[j] = e;
    }
}
__global__ __launch_bounds__(256) void fork_rows_kernel(ForkArgs a) { fork_rows(a, blockIdx.x, threadIdx.x, 256); }

// Plan: one thread per pair; with `rows` (few pairs and entries) the new rows in the same launch, a wave per pair. Pages of old
// rows are released by the last launch, so pages given out here are never ones that a copy still reads.
// Bound by latency (references, sums, list, rows: dependent round trips of one work-group): 6 to 7 us for 8 pairs of 32 pages.
__global__ __launch_bounds__(PLAN_T) void fork_plan_kernel(ForkArgs a, int rows) {
    __shared__ int tmp[PLAN_T / 64];
    __shared__ int sdst[MAX_SEQS];
    const int i = threadIdx.x;
    const int d = i < a.M ? a.dst[i] : -1, s = i < a.M ? a.src[i] : -1;
    sdst[i] = d;
    __syncthreads();
    bool valid = i < a.M && d >= 0 && d < a.B && s < a.B;
    if (valid)
        for (int j = 0; j < i; ++j) valid = valid && sdst[j] != d;  // (the first pair of a place counts)
    int n = 0, need = 0, copies = 0;
    if (valid) {
        n = s < 0 ? 0 : clamp_len(a.length[s], a.W, a.lt);
        const int64_t total = (int64_t(n) + a.room + a.T - 1) >> a.lt;
        const int full = n >> a.lt, used = (n + a.T - 1) >> a.lt;
        if (total > a.W) {
            valid = false;
        } else if (s == d) {  // a sequence that stays: only the pages of its room
            for (int j = full; j < int(total); ++j) need += uint32_t(a.table[d * a.ts + j]) >= uint32_t(a.P);
        } else {
            need = int(total) - (a.share ? full : 0);
            copies = a.share ? used - full : used;
        }
    }
    if (!valid) n = need = copies = 0;
    int want = 0, all = 0, upto = 0, have = 0, cend = 0;
    if (__syncthreads_or(need)) {
        upto = block_sum_incl(need, tmp, want);
        have = free_pages(a.refs, a.P, want, a.fresh, tmp);
    }
    const bool served = valid && (need == 0 || upto <= have);  // (a drop frees pages: it waits for none)
    if (__syncthreads_or(served ? copies : 0)) cend = block_sum_incl(served ? copies : 0, tmp, all);
    if (i < a.M) {
        reinterpret_cast<int4*>(a.pair)[i] = make_int4(valid ? (served ? 1 : 0) : -1, n, upto - need, cend - copies);
        a.status[i] = valid ? (served ? 1 : 0) : -1;
    }
    if (i == 0) a.head[0] = all;
    if (!rows) return;  // (uniform)
    __syncthreads();
    for (int x = i >> 6; x < a.M; x += PLAN_T / 64) fork_rows(a, x, i & 63, 64);
}

// The copies (work-groups past the pairs', in pieces of 16 KiB) and, by the first `pairs` work-groups, what the call
// changes in the tables: the old rows' references given back, the new rows, lengths and slots.
// Bound by the bytes: 16 bytes per lane and load, four loads in flight per wave. 66 pages of 4 MiB: 130 us a call, 4.3 TB/s
// read and written together (4.8 in one large copy).
constexpr int PIECE = 256 * 16 * 4;
__device__ __forceinline__ void copy_piece(const unsigned char* from, unsigned char* to, int64_t bytes) {
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t o = (int64_t(k) * 256 + threadIdx.x) * 16;
        if (o < bytes) v[k] = *reinterpret_cast<const u32x4*>(from + o);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t o = (int64_t(k) * 256 + threadIdx.x) * 16;
        if (o < bytes) *reinterpret_cast<u32x4*>(to + o) = v[k];
    }
}

__global__ __launch_bounds__(256) void fork_copy_kernel(ForkArgs a) {
    if (int(blockIdx.x) < a.M) {
        const int i = blockIdx.x;
        const int4 p = reinterpret_cast<const int4*>(a.pair)[i];
        const int32_t* row = a.rows + int64_t(i) * a.W;
        if (p.x == 1) {
            const int d = a.dst[i], s = a.src[i];
            for (int j = threadIdx.x; j < a.W; j += 256) {
                const int old = a.table[d * a.ts + j];
                if (s != d && old >= 0 && old < a.P) atomicSub(a.refs + old, 1);
                a.table[d * a.ts + j] = row[j];
            }
            if (threadIdx.x == 0) a.length[d] = p.y;
        }
        if (a.slots)
            for (int r = threadIdx.x; r < a.room; r += 256) {
                const int64_t t = int64_t(p.y) + r;
                const int e = p.x == 1 ? row[t >> a.lt] : -1;
                a.slots[int64_t(i) * a.room + r] = e >= 0 ? (int64_t(e) << a.lt) + (t & (a.T - 1)) : -1;
            }
        return;
    }
    const int pieces = int((a.page_bytes + PIECE - 1) / PIECE), sums = a.share || !a.ksum ? 0 : a.sum_chunks;
    const int64_t jobs = int64_t(a.head[0]) * (int64_t(a.chunks) * pieces + sums);
    const int64_t per = int64_t(a.chunks) * pieces;
    for (int64_t job = int64_t(blockIdx.x) - a.M; job < jobs; job += int64_t(gridDim.x) - a.M) {
        const int c = int(job / (per + sums));
        const int64_t in = job % (per + sums);
        const int2 pg = a.copies[c];
        if (pg.x < 0) continue;
        if (in < per) {
            const int64_t chunk = in / pieces, o = in % pieces * PIECE;
            unsigned char* base = a.kv + chunk * a.P * a.page_bytes + o;
            copy_piece(base + pg.x * a.page_bytes, base + pg.y * a.page_bytes, a.page_bytes - o);
        } else {
            unsigned char* base = a.ksum + (in - per) * a.P * a.sum_bytes;
            copy_piece(base + pg.x * a.sum_bytes, base + pg.y * a.sum_bytes, a.sum_bytes);
        }
    }
}

// ---- page_commit ----------------------------------------------------------------------------------------
struct CommitArgs {
    unsigned char* kv;
    uint16_t* ksum;  // null: none
    int32_t* table;
    int64_t ts;
    const int32_t* length;
    int32_t* new_length;
    int32_t* refs;
    const int32_t* count;
    const int32_t* path;  // [B][R] or null
    int64_t* slots;       // [B][room] or null
    int32_t* status;
    int B, W, P, T, lt, D, L, Hk, R, room, half;  // half: fp16 elements, else bf16
    int per_wg, wgs;      // chunks a work-group of the move takes, and such work-groups per sequence
    int32_t* fresh;
};

__device__ __forceinline__ int page_at(const CommitArgs& a, int b, int64_t t) {
    const int64_t j = t >> a.lt;
    const int e = j < a.W ? a.table[b * a.ts + j] : -1;
    return e >= 0 && e < a.P ? e : -1;
}

__device__ __forceinline__ bool commit_fits(const CommitArgs& a, int n, int c) {
    return c >= 0 && n >= 0 && !(a.path && c > a.R) && int64_t(n) + c <= int64_t(a.W) << a.lt;
}

// Sequence b's rows n + path[k] to n + k, and the mean keys of the pages that fill, for the chunks from c0. The work-group
// holds every row of its chunks in registers before it writes one, so no order among the rows matters; chunks do not meet.
// Bound by latency (dependent round trips), hence many work-groups: 32 sequences of 8 rows over 128 chunks are 256.
__device__ void commit_move(const CommitArgs& a, int b, int c0) {
    __shared__ int64_t from[MAX_PATH], to[MAX_PATH];
    __shared__ int bad;
    const int n = a.length[b], c = a.count[b], t = threadIdx.x;
    if (!commit_fits(a, n, c)) return;  // (uniform)
    if (t == 0) bad = 0;
    __syncthreads();
    const int j0 = n >> a.lt, j1 = (n + c + a.T - 1) >> a.lt;
    if (t < c) {
        const int32_t* path = a.path + int64_t(b) * a.R;
        const int k = path[t], before = t ? path[t - 1] : -1;
        const int p = k >= 0 && k < a.R ? page_at(a, b, int64_t(n) + k) : -1, q = page_at(a, b, int64_t(n) + t);
        from[t] = k == t ? -1 : (int64_t(p) << a.lt) + ((n + k) & (a.T - 1));
        to[t] = (int64_t(q) << a.lt) + ((n + t) & (a.T - 1));
        if (k <= before || p < 0 || q < 0) bad = 1;
    }
    if (t >= MAX_PATH && t - MAX_PATH < j1 - j0 && page_at(a, b, int64_t(j0 + t - MAX_PATH) << a.lt) < 0) bad = 1;
    __syncthreads();
    if (bad) return;
    const int lanes = a.D / 8, items = c * lanes;  // 16-byte pieces of a chunk's rows
    const int chunks = a.L * 2 * a.Hk, mine = min(a.per_wg, chunks - c0), live = mine * items;
    constexpr int MOST = 2;  // 64 rows of 32 pieces
    u32x4 v[MOST];
    const int64_t chunk_bytes = (int64_t(a.P) << a.lt) * a.D * 2;
    auto place = [&](int x, const int64_t* rows) -> unsigned char* {
        const int in = x % items, k = in / lanes;
        return from[k] < 0 ? nullptr : a.kv + (c0 + x / items) * chunk_bytes + rows[k] * a.D * 2 + in % lanes * 16;
    };
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int x = i * PLAN_T + t;
        unsigned char* p = x < live ? place(x, from) : nullptr;
        if (p) v[i] = *reinterpret_cast<const u32x4*>(p);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int x = i * PLAN_T + t;
        unsigned char* p = x < live ? place(x, to) : nullptr;
        if (p) *reinterpret_cast<u32x4*>(p) = v[i];
    }
    const int filled = ((n + c) >> a.lt) - j0;
    if (!a.ksum || filled == 0) return;
    __syncthreads();  // (the rows above, read by other waves)
    for (int x = t >> 6; x < filled * mine; x += PLAN_T / 64) {
        const int chunk = c0 + x % mine, kc = chunk / (2 * a.Hk) * a.Hk + chunk % (2 * a.Hk);
        if (chunk % (2 * a.Hk) >= a.Hk) continue;  // (values)
        mean_key(a, kc, page_at(a, b, int64_t(j0 + x / mine) << a.lt), t & 63);
    }
}

// Mean keys of the pages that a commit without a path fills, one wave per (page, layer, kv head). The pages of all sequences
// are numbered through (their counts summed in every work-group), so a batch of short tails and one long prompt spread
// alike. Bound by the bytes of the keys.
__device__ void commit_sums(const CommitArgs& a, int block, int blocks) {
    __shared__ int upto[MAX_SEQS], first[MAX_SEQS], tmp[PLAN_T / 64];  // pages filled in sequences 0..b, their first
    const int t = threadIdx.x;
    int f = 0;
    if (t < a.B) {
        const int n = a.length[t], c = a.count[t];
        first[t] = n >> a.lt;
        if (commit_fits(a, n, c)) f = ((n + c) >> a.lt) - (n >> a.lt);
    }
    int total;
    upto[t] = block_sum_incl(f, tmp, total);
    __syncthreads();
    const int64_t keys = int64_t(a.L) * a.Hk, jobs = total * keys;
    for (int64_t job = int64_t(block) * (PLAN_T / 64) + (t >> 6); job < jobs; job += int64_t(blocks) * (PLAN_T / 64)) {
        const int page_no = int(job / keys);
        int lo = 0, hi = a.B - 1;  // the sequence: the first whose sum passes page_no
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] > page_no) hi = mid;
            else lo = mid + 1;
        }
        const int e = page_at(a, lo, int64_t(first[lo] + page_no - (lo ? upto[lo - 1] : 0)) << a.lt);
        if (e >= 0) mean_key(a, job % keys, e, t & 63);
    }
}

// Lengths, pages for the next rows and their slots: one thread per sequence (a span of many entries by a whole wave).
__device__ void commit_plan(const CommitArgs& a) {
    __shared__ int tmp[PLAN_T / 64], ends[MAX_SEQS], bad[MAX_SEQS];
    const int b = threadIdx.x, lane = b & 63;
    const int n = b < a.B ? a.length[b] : -1, c = b < a.B ? a.count[b] : 0;
    bad[b] = 0;
    ends[b] = n;
    bool valid = b < a.B && commit_fits(a, n, c);
    int64_t total = 0;
    bool narrow = false;  // (room past the table's width gets no page)
    if (valid) {
        total = (int64_t(n) + c + a.room + a.T - 1) >> a.lt;
        narrow = total > a.W;
        if (narrow) total = a.W;
    }
    // the committed rows' entries have to be pages; missing ones behind them are given
    const int j0 = n >> a.lt, j1 = valid ? (n + c + a.T - 1) >> a.lt : 0, j2 = int(total);
    int need = 0, holes = 0;
    const bool wide = valid && j2 - j0 > 8;
    if (valid && !wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = j0 + i;
            const bool miss = j < j2 && page_at(a, b, int64_t(j) << a.lt) < 0;
            holes += miss && j < j1;
            need += miss && j >= j1;
        }
    }
    if (a.path) {  // the checks of the move, a thread per row
        __syncthreads();
        for (int x = b; x < a.B * a.R; x += PLAN_T) {
            const int q = x / a.R, k = x % a.R, cq = a.count[q], nq = ends[q];
            if (!commit_fits(a, nq, cq) || k >= cq) continue;
            const int p = a.path[x], before = k ? a.path[x - 1] : -1;
            if (p <= before || p >= a.R || page_at(a, q, int64_t(nq) + p) < 0) bad[q] = 1;
        }
        __syncthreads();
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(wide);
    while (todo) {  // (uniform in the wave)
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int bb = __builtin_amdgcn_readlane(b, l), x0 = __builtin_amdgcn_readlane(j0, l), x1 = __builtin_amdgcn_readlane(j1, l),
                  x2 = __builtin_amdgcn_readlane(j2, l);
        int in = 0, behind = 0;
#pragma unroll 4
        for (int j = x0 + lane; j < x2; j += 64) {
            const bool miss = page_at(a, bb, int64_t(j) << a.lt) < 0;
            in += miss && j < x1;
            behind += miss && j >= x1;
        }
        for (int d = 32; d; d >>= 1) {
            in += __shfl_xor(in, d, 64);
            behind += __shfl_xor(behind, d, 64);
        }
        if (lane == l) {
            holes = in;
            need = behind;
        }
    }
    valid = valid && holes == 0 && bad[b] == 0;
    if (!valid) need = 0;
    int upto = 0, have = 0;
    if (__syncthreads_or(need)) {  // (most steps stay in their pages)
        int want;
        upto = block_sum_incl(need, tmp, want);
        have = free_pages(a.refs, a.P, want, a.fresh, tmp);
        __syncthreads();  // (the list, written by other threads)
    }
    const bool served = valid && (need == 0 || upto <= have);
    if (served && need && !wide) {
        int at = upto - need;
        for (int j = j1; j < j2; ++j)
            if (page_at(a, b, int64_t(j) << a.lt) < 0) {
                const int e = a.fresh[at++];
                a.table[b * a.ts + j] = e;
                a.refs[e] = 1;
            }
    }
    todo = __builtin_amdgcn_ballot_w64(wide && served && need);
    while (todo) {  // (uniform in the wave)
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int bb = __builtin_amdgcn_readlane(b, l), x1 = __builtin_amdgcn_readlane(j1, l), x2 = __builtin_amdgcn_readlane(j2, l);
        int at = __builtin_amdgcn_readlane(upto - need, l);
        for (int k0 = x1; k0 < x2; k0 += 64) {
            const int j = k0 + lane;
            const bool miss = j < x2 && page_at(a, bb, int64_t(j) << a.lt) < 0;
            const uint64_t m = __builtin_amdgcn_ballot_w64(miss);
            if (miss) {
                const int e = a.fresh[at + __popcll(m & ((uint64_t(1) << lane) - 1))];
                a.table[bb * a.ts + j] = e;
                a.refs[e] = 1;
            }
            at += __popcll(m);
        }
    }
    ends[b] = valid ? n + c : -1;
    if (b < a.B) {
        a.status[b] = valid ? (served && !narrow ? 1 : 0) : (c < 0 ? 1 : -1);
        a.new_length[b] = valid ? n + c : n;
    }
    if (!a.slots) return;
    __syncthreads();  // (ends, and the entries given above)
    for (int x = b; x < a.B * a.room; x += PLAN_T) {
        const int q = x / a.room;
        const int64_t t = int64_t(ends[q]) + x % a.room;
        const int e = ends[q] >= 0 ? page_at(a, q, t) : -1;
        a.slots[x] = e >= 0 ? (int64_t(e) << a.lt) + (t & (a.T - 1)) : -1;
    }
}

// The plan (`plans` work-groups, 1 or 0) and the moves and means, in one launch where the new lengths go elsewhere than the
// old ones. They do not meet: the plan changes entries behind the committed rows' alone, of sequences whose rows all have
// pages already, and each checks a sequence alike.
__global__ __launch_bounds__(PLAN_T) void commit_kernel(CommitArgs a, int plans) {
    const int x = int(blockIdx.x) - plans;
    if (x < 0) commit_plan(a);
    else if (a.path) commit_move(a, x / a.wgs, x % a.wgs * a.per_wg);
    else commit_sums(a, x, int(gridDim.x) - plans);
}

// ints of the fork's workspace ahead of the copies: head, pairs, fresh pages, rows
int64_t fork_ints(int64_t M, int64_t W) { return 4 + 4 * M + M * W + M * W; }

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_page_fork_workspace(int64_t pairs, int64_t W) {
    if (pairs < 1 || pairs > MAX_SEQS || W < 1 || W > (int64_t(1) << 26)) return 0;
    return size_t((fork_ints(pairs, W) + 3) / 4 * 4) * 4 + size_t(pairs) * W * sizeof(int2);
}

extern "C" int mdx_page_fork(void* kv, void* ksum, int64_t L, int64_t Hk, int64_t P, int64_t T, int64_t D, int32_t* table,
                             int64_t table_stride, int64_t B, int64_t W, int32_t* length, int32_t* refs, const int32_t* dst,
                             const int32_t* src, int64_t pairs, int64_t room, int32_t share, int64_t* slots, int32_t* status,
                             void* workspace, size_t workspace_bytes, void* stream) {
    MDX_CHECK(kv && table && length && refs && dst && src && status, "null pointer");
    const int lt = log2_of(T);
    MDX_CHECK(lt >= 0, "page rows: a power of two in 16..1024");
    MDX_CHECK(L >= 1 && Hk >= 1 && P >= 1 && L * Hk <= 65536 && P <= (int64_t(1) << 30) && D >= 8 && D <= 1024 && D % 8 == 0,
              "layers, heads, pages, head_dim (a multiple of 8)");
    MDX_CHECK(B >= 1 && B <= (int64_t(1) << 24) && W >= 1 && (W << lt) < (int64_t(1) << 30) && table_stride >= W && table_stride <= (int64_t(1) << 26),
              "table [sequences, W], under 2^30 tokens a sequence");
    MDX_CHECK(pairs >= 1 && pairs <= MAX_SEQS && room >= 0 && room < (int64_t(1) << 30), "1..1024 pairs, room");
    MDX_CHECK(pairs * W < (int64_t(1) << 30), "too many pairs times table entries");
    MDX_CHECK(aligned(kv, 16) && aligned(ksum, 16), "16-byte aligned cache");
    MDX_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= mdx_page_fork_workspace(pairs, W),
              "workspace: %zu bytes, 16-byte aligned", mdx_page_fork_workspace(pairs, W));
    ForkArgs a{};
    a.kv = static_cast<unsigned char*>(kv);
    a.ksum = static_cast<unsigned char*>(ksum);
    a.page_bytes = T * D * 2;
    a.sum_bytes = D * 2;
    a.chunks = int(L * 2 * Hk);
    a.sum_chunks = int(L * Hk);
    a.table = table;
    a.ts = table_stride;
    a.length = length;
    a.refs = refs;
    a.dst = dst;
    a.src = src;
    a.slots = slots;
    a.status = status;
    a.B = int(B), a.W = int(W), a.P = int(P), a.T = int(T), a.lt = lt, a.M = int(pairs), a.room = int(room), a.share = share;
    a.head = static_cast<int32_t*>(workspace);
    a.pair = a.head + 4;
    a.fresh = a.pair + 4 * pairs;
    a.rows = a.fresh + pairs * W;
    a.copies = reinterpret_cast<int2*>(a.head + (fork_ints(pairs, W) + 3) / 4 * 4);
    hipStream_t st = static_cast<hipStream_t>(stream);
    // (the planning work-group builds the rows too: 512 entries 9.8 us a call, 12.3 with a launch for them; 4096: 14.0 and 12.8;
    // 8192: 20.2 and 14.6)
    const bool few = pairs * W <= 2048;
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(PLAN_T), 0, st, a, few ? 1 : 0);
    MDX_LAUNCHED();
    if (!few) {
        hipLaunchKernelGGL(fork_rows_kernel, dim3(unsigned(pairs)), dim3(256), 0, st, a);
        MDX_LAUNCHED();
    }
    hipLaunchKernelGGL(fork_copy_kernel, dim3(unsigned(pairs + 2048)), dim3(256), 0, st, a);
    MDX_LAUNCHED();
    return MDX_OK;
}

extern "C" size_t mdx_page_commit_workspace(int64_t B, int64_t W) {
    if (B < 1 || B > MAX_SEQS || W < 1 || W > (int64_t(1) << 26)) return 0;
    return size_t(B * W) * 4;
}

extern "C" int mdx_page_commit(void* kv, void* ksum, int32_t dtype, int64_t L, int64_t Hk, int64_t P, int64_t T, int64_t D,
                               int32_t* table, int64_t table_stride, int64_t B, int64_t W, const int32_t* length,
                               int32_t* new_length, int32_t* refs, const int32_t* count, const int32_t* path, int64_t R,
                               int64_t room, int64_t* slots, int32_t* status, void* workspace, size_t workspace_bytes,
                               void* stream) {
    MDX_CHECK(kv && table && length && new_length && refs && count && status, "null pointer");
    MDX_CHECK(dtype == MDX_DT_BF16 || dtype == MDX_DT_F16, "bf16 or fp16");
    const int lt = log2_of(T);
    MDX_CHECK(lt >= 0, "page rows: a power of two in 16..1024");
    MDX_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
    MDX_CHECK(L >= 1 && Hk >= 1 && P >= 1 && L * Hk <= 65536 && P <= (int64_t(1) << 30), "layers, heads, pages");
    MDX_CHECK(B >= 1 && B <= MAX_SEQS && W >= 1 && (W << lt) < (int64_t(1) << 30) && table_stride >= W && table_stride <= (int64_t(1) << 26),
              "table [1..1024 sequences, W], under 2^30 tokens a sequence");
    MDX_CHECK(B * W < (int64_t(1) << 30), "too many sequences times table entries");
    MDX_CHECK(new_length == length || new_length + B <= length || length + B <= new_length, "new_length: length itself, or apart from it");
    MDX_CHECK(!path || (R >= 1 && R <= MAX_PATH), "a path has 1..64 rows");
    MDX_CHECK(room >= 0 && room <= 65536 && B * room < (int64_t(1) << 30), "room 0..65536");
    MDX_CHECK(aligned(kv, 16) && aligned(ksum, 16), "16-byte aligned cache");
    MDX_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= mdx_page_commit_workspace(B, W),
              "workspace: %zu bytes, 16-byte aligned", mdx_page_commit_workspace(B, W));
    CommitArgs a{};
    a.kv = static_cast<unsigned char*>(kv);
    a.ksum = static_cast<uint16_t*>(ksum);
    a.table = table;
    a.ts = table_stride;
    a.length = length;
    a.new_length = new_length;
    a.refs = refs;
    a.count = count;
    a.path = path;
    a.slots = slots;
    a.status = status;
    a.B = int(B), a.W = int(W), a.P = int(P), a.T = int(T), a.lt = lt, a.D = int(D), a.L = int(L), a.Hk = int(Hk);
    a.R = int(path ? R : 0), a.room = int(room), a.half = dtype == MDX_DT_F16;
    a.fresh = static_cast<int32_t*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t chunks = L * 2 * Hk;
    // chunks per work-group of the move: 2048 pieces of 16 bytes (two in flight per thread)
    const int64_t items = (path ? R : 1) * D / 8;
    a.per_wg = int(2048 / items);
    a.wgs = int((chunks + a.per_wg - 1) / a.per_wg);
    const int64_t work = path ? B * a.wgs : ksum ? 256 : 0;
    MDX_CHECK(work < (int64_t(1) << 30), "too many chunks times sequences");
    if (work && new_length == length) {
        hipLaunchKernelGGL(commit_kernel, dim3(unsigned(work)), dim3(PLAN_T), 0, st, a, 0);
        MDX_LAUNCHED();
        hipLaunchKernelGGL(commit_kernel, dim3(1), dim3(PLAN_T), 0, st, a, 1);
    } else {
        hipLaunchKernelGGL(commit_kernel, dim3(unsigned(1 + work)), dim3(PLAN_T), 0, st, a, 1);
    }
    MDX_LAUNCHED();
    return MDX_OK;
}
