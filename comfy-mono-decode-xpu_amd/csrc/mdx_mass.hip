// The attention weight that cached tokens draw, summed up (mdx_attn_mass): what an eviction goes by (mdx_page_evict).
//
// out[b][g][t] = (t < n ? prior[b][g][t] : 0) + sum over rows k < count[b] that attend t and the heads h of kv head g of
// exp(scale q[b][path[b][k]][h] . key_t - lse[b][path[b][k]][h]); row k attends the tokens t <= n + k (n = length[b]; a row's own
// place is n + k), of these the first `sinks` and the last `window`. lse is the rows' log-sum-exp of mdx_attn_window, so a
// weight needs nothing but its own score: the keys are read once and no token waits for another.
//
// S^T = K Q^T by v_mfma_f32_16x16x32 (A: 16 tokens x 32 dims, B: 16 query rows, the lane holds scores of one row and four
// tokens), keys straight from the pages to registers (16 bytes per lane and load, whole 64-byte pieces of 16 tokens), one
// exponential per score, fp32 sums per token in the lane, joined over the 16 rows' lanes at the end by exchanges that halve the
// values (45 instructions for 64 tokens instead of 64 sums). A token's sum is one wave's (or a work-group's waves', joined in their
// order): no atomics, the same bits every time. What a row does not attend is selected out, not multiplied: non-finite keys
// there do not reach it.
//
// Few rows: a wave per 16 TT tokens, bound by the keys' bytes (single tokens of 32 sequences of up to 8191, 8 kv heads of 128: 61 us
// at 4.9 TB/s). Many rows (below): bound by the exponentials and the matrix instructions in about equal parts (1000 rows of 32
// heads over 4000 tokens: 62 us, 0.6 PFLOP/s).
//
// Reference: none (its cache is never thinned).
#include <limits.h>

#include <atomic>

#include "mdx_lds.hpp"

namespace mdx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct Fp16 {
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

struct MassArgs {
    const uint16_t* q;  // [B, S, H, D], strides qb, qs, qh
    int64_t qb, qs, qh;
    const uint16_t* key;  // [Hk, P, T, D], strides kh, kp, kt
    int64_t kh, kp, kt;
    const int32_t* table;  // [B, W], row stride ts
    int64_t ts;
    const int32_t* length;  // [B]
    const float* lse;       // [B, S, H]
    const float* prior;     // [B, Hk, N], strides pb, ph; null: zeros
    int64_t pb, ph;
    const int32_t* count;  // [B] or null (S)
    const int32_t* path;   // [B, S] or null (row k is k)
    float* out;            // [B, Hk, N], strides ob, oh
    int64_t ob, oh;
    int B, S, H, Hk, G, W, P, lt, N;
    int window, sinks;
    int tiles;  // runs of tokens that the grid covers at once
    int shares;   // work-groups that share the rows of a run (MANY rows)
    float* part;  // [shares][B][Hk][tiles * run]: their sums, where there are several
    float zs;   // scale * log2(e)
};

// the sums of 16 (V = 16) or 8 values over a row of 16 lanes: lane c16 receives value c16 (V = 8: value c16 % 8)
template <int CTRL>
__device__ __forceinline__ float other(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int N, int CTRL>
__device__ __forceinline__ void halve(float* v, bool up) {  // (the partner across has the other half's sums)
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float keep = up ? v[j + N] : v[j], give = up ? v[j] : v[j + N];
        v[j] = keep + other<CTRL>(give);
    }
}
constexpr int ROR8 = 0x128, HALF_MIRROR = 0x141, QUAD_REVERSE = 0x1B, QUAD_SWAP = 0xB1;  // lane ^ 8, ^ 7, ^ 3, ^ 1
template <int V>
__device__ __forceinline__ float row_sums(float* v, int c16) {
    if constexpr (V == 16) {
        halve<8, ROR8>(v, c16 & 8);
    } else {
        static_assert(V == 8, "");
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += other<ROR8>(v[j]);
    }
    halve<4, HALF_MIRROR>(v, c16 & 4);
    halve<2, QUAD_REVERSE>(v, c16 & 2);
    halve<1, QUAD_SWAP>(v, c16 & 1);
    return v[0];
}

typedef __attribute__((address_space(4))) const int32_t* const_i32p;
__device__ __forceinline__ int uload(const int32_t* p) { return *(const_i32p)(p); }  // (a scalar load: uniform addresses)

// TT tiles of 16 tokens per wave; SPLIT: the four waves of the work-group share them and take the row tiles in turn; PATH: the
// rows go by a.path.
template <class E, int D, int TT, bool SPLIT, bool PATH>
__global__ __launch_bounds__(256, 3) void attn_mass_kernel(MassArgs a) {
    constexpr int KK = D / 32, TOK = 16 * TT, RUN = SPLIT ? TOK : 4 * TOK;
    static_assert(TT == 2 || TT == 4, "");
    __shared__ float part[SPLIT ? 4 : 1][TOK];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
    // (kv heads in turn: an XCD's work-groups share the queries of one)
    const int kh = int(blockIdx.x) % a.Hk, rest = int(blockIdx.x) / a.Hk, b = rest / a.tiles;
    const int n = max(0, min(uload(a.length + b), a.W << a.lt));
    const int rows = a.count ? max(0, min(uload(a.count + b), a.S)) : a.S;
    const int end = min(min(n + rows, a.W << a.lt), a.N);
    const int32_t* trow = a.table + b * a.ts;
    const float* lse = a.lse + int64_t(b) * a.S * a.H + kh * a.G;
    const uint16_t* queries = a.q + b * a.qb + kh * a.G * a.qh + 8 * g;
    const int32_t* path = PATH ? a.path + int64_t(b) * a.S : nullptr;
    constexpr int STEP = SPLIT ? 4 : 1;  // a wave's row tiles are so far apart
    const int step_k = 16 * STEP / a.G, step_h = 16 * STEP % a.G;
    const int64_t q_step = step_k * a.qs + step_h * a.qh, q_over = q_step + a.qs - a.G * a.qh;
    for (int run = rest % a.tiles; run * RUN < end; run += a.tiles) {
        const int t0 = run * RUN + (SPLIT ? 0 : w * TOK);
        if (!SPLIT && t0 >= end) continue;
        // ---- row tiles that can attend a token of the run: rows k from t0 - n on, and in a window up to the last token's
        const int k_first = max(0, t0 - n);
        const int64_t k_last = t0 < a.sinks ? rows - 1 : min(int64_t(rows) - 1, int64_t(t0) + TOK - 2 - n + a.window);
        const int r_first = k_first * a.G / 16 + (SPLIT ? w : 0), r_end = k_last < k_first ? 0 : int((k_last + 1) * a.G + 15) / 16;
        f32x4 sum[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (r_first < r_end) {  // (uniform in the wave)
            // ---- a tile's queries and log-sum-exps, one tile ahead of their use
            struct Rows {
                u32x4 q[KK];
                float base;  // its log-sum-exp, as loaded: its first use waits for it, a tile later
                int k;       // -1: no row
            };
            const int r0 = r_first * 16 + c16;
            int k_at = r0 / a.G, h_at = r0 % a.G;
            const uint16_t* q_at = queries + k_at * a.qs + h_at * a.qh;  // (without a path: row k's queries, advanced by sums)
            auto fetch = [&]() {
                Rows x;
                bool live = k_at < rows;
                int s = live ? k_at : 0;
                const uint16_t* src = live ? q_at : queries;
                int h = live ? h_at : 0;
                if constexpr (PATH) {
                    s = path[s];
                    live = live && uint32_t(s) < uint32_t(a.S);
                    s = live ? s : 0;
                    src = queries + s * a.qs + h * a.qh;
                }
                x.base = lse[uint32_t(s) * uint32_t(a.H) + uint32_t(h)];
                x.k = live ? k_at : -1;
#pragma unroll
                for (int i = 0; i < KK; ++i) x.q[i] = *reinterpret_cast<const u32x4*>(src + 32 * i);
                h_at += step_h;
                const bool over = h_at >= a.G;
                h_at -= over ? a.G : 0;
                k_at += step_k + (over ? 1 : 0);
                q_at += over ? q_over : q_step;
                return x;
            };
            Rows next = fetch();
            // ---- the tokens' keys, as A operands
            u32x4 kf[TT][KK];
            uint32_t there = 0;  // tiles that stand in a page
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                const int t = t0 + 16 * i, e = t < end ? uload(trow + (t >> a.lt)) : -1;
                const bool in = uint32_t(e) < uint32_t(a.P);
                there |= in ? 1u << i : 0u;
                // (a tile without a page reads the pool's first rows: in bounds, and selected out)
                const uint16_t* src = a.key + kh * a.kh + (in ? int64_t(e) * a.kp + int64_t(t & ((1 << a.lt) - 1)) * a.kt : 0) + c16 * a.kt + 8 * g;
#pragma unroll
                for (int k = 0; k < KK; ++k) kf[i][k] = *reinterpret_cast<const u32x4*>(src + 32 * k);
            }
            // they have arrived before the loop: the waits for them in it would be for the next tile's queries too
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int k = 0; k < KK; ++k) asm volatile("" : "+v"(kf[i][k]));
            // Row tiles in which every row attends every token of the run: k >= the last token's own row, and in a window k up to
            // the first token's last one.
            const int all_k = t0 + TOK - 1 - n;
            const int64_t near_k = int64_t(t0) - n - 1 + a.window;
            const int whole_from = there != (1u << TT) - 1u ? INT_MAX : all_k <= 0 ? 0 : (all_k * a.G + 15) / 16;
            const int whole_end = t0 + TOK <= a.sinks ? INT_MAX : int(min(int64_t(INT_MAX), (near_k + 1) * a.G) >> 4);
            uint64_t pages = 0;  // tokens of the run that stand in pages
#pragma unroll
            for (int i = 0; i < TT; ++i) pages |= (there >> i) & 1u ? uint64_t(0xFFFF) << (16 * i) : 0;
            auto scores = [&](const Rows& x, f32x4 (&z)[TT]) {
#pragma unroll
                for (int i = 0; i < TT; ++i) z[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KK; ++k)
#pragma unroll
                    for (int i = 0; i < TT; ++i) z[i] = E::mfma(kf[i][k], x.q[k], z[i]);
            };
            for (int rt = r_first; rt < r_end; rt += STEP) {
                const Rows row = next;
                if (rt + STEP < r_end) next = fetch();
                f32x4 z[TT];
                scores(row, z);
                // (+inf: the row gives nothing)
                const float sub = row.k >= 0 && row.base > -INFINITY ? row.base * 1.44269504088896340736f : INFINITY;
                if (rt >= whole_from && rt < whole_end && __builtin_amdgcn_ballot_w64(sub == INFINITY) == 0) {  // (uniform)
#pragma unroll
                    for (int i = 0; i < TT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[i][e] += __builtin_amdgcn_exp2f(fmaf(z[i][e], a.zs, -sub));
                } else {
                    // the run's tokens that this row attends: t < lim, of these t < sinks or t >= lim - window
                    const int lim = n + row.k + 1 - t0, lo = lim - a.window, f = a.sinks - t0;
                    auto below = [](int m) -> uint64_t { return m <= 0 ? 0 : m >= 64 ? ~uint64_t(0) : (uint64_t(1) << m) - 1; };
                    uint64_t in = sub == INFINITY ? 0 : below(lim) & (below(f) | ~below(lo)) & pages;
                    in >>= 4 * g;
#pragma unroll
                    for (int i = 0; i < TT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p = __builtin_amdgcn_exp2f(fmaf(z[i][e], a.zs, -sub));
                            sum[i][e] += (in >> (16 * i + e)) & 1 ? p : 0.f;
                        }
                }
            }
        }
        float v[4 * TT];
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = sum[i][e];
        const float mine = row_sums<4 * TT>(v, c16);
        const int token = 16 * ((c16 % (4 * TT)) >> 2) + 4 * g + (c16 & 3);
        auto put = [&](int t, float x) {
            if (t >= end) return;
            const float p = t < n && a.prior ? a.prior[b * a.pb + kh * a.ph + t] : 0.f;
            a.out[b * a.ob + kh * a.oh + t] = p + x;
        };
        if constexpr (SPLIT) {
            if (c16 < 4 * TT) part[w][token] = mine;
            __syncthreads();
            if (threadIdx.x < TOK)
                put(t0 + int(threadIdx.x), (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]));
            __syncthreads();
        } else {
            if (c16 < 4 * TT) put(t0 + token, mine);
        }
    }
}

// ---- many rows --------------------------------------------------------------------------------------------------
// The four waves of a work-group hold 16 TT tokens each and go through the same rows, which come to LDS by direct loads, a ring
// of three stages of 16 KiB (each wave reading them from L2 for itself: 1000 rows over 4000 tokens 93 us, at 7 TB/s out of L2). The
// rows of a run are shared out to several work-groups where there are few runs; a second launch then joins their sums.
template <int D>
struct Many {
    static constexpr int TT = D == 256 ? 2 : 4, TOK = 16 * TT, RUN = 4 * TOK;  // tokens of a wave, of a work-group
    static constexpr int RB = 2 * D, SR = 16384 / RB, NS = 3;                   // bytes of a row, rows of a stage, stages
    static constexpr int RPL = 1024 / RB, LPR = 64 / RPL, WR = SR / 4;          // rows and lanes a row of a direct load, rows a wave loads
    static constexpr int LSE = 4 * 64 * 4;                                      // bytes of a stage's log-sum-exps: WR of each 64
    static constexpr int LDS = NS * (16384 + LSE);
};

template <class E, int D>
__global__ __launch_bounds__(256, 3) void attn_mass_many_kernel(MassArgs a) {
    using M = Many<D>;
    constexpr int KK = D / 32, TT = M::TT, TOK = M::TOK, RUN = M::RUN, SR = M::SR, NS = M::NS, WR = M::WR, LOADS = 5;
    extern __shared__ __align__(256) unsigned char smem[];  // [NS] stages of rows, then [NS] of log-sum-exps
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
    const int share = int(blockIdx.x) % a.shares, x0 = int(blockIdx.x) / a.shares;
    const int kh = x0 % a.Hk, rest = x0 / a.Hk, b = rest / a.tiles;
    const int n = max(0, min(uload(a.length + b), a.W << a.lt));
    const int rows = a.count ? max(0, min(uload(a.count + b), a.S)) : a.S;
    const int end = min(min(n + rows, a.W << a.lt), a.N);
    const int32_t* trow = a.table + b * a.ts;
    const uint32_t ring = lds_addr(smem), lse_ring = ring + NS * 16384;
    const uint16_t* queries = a.q + b * a.qb + kh * a.G * a.qh;
    const float* lse = a.lse + int64_t(b) * a.S * a.H + kh * a.G;
    const int step_k = SR / a.G, step_h = SR % a.G, all_rows = rows * a.G;
    const int64_t q_step = step_k * a.qs + step_h * a.qh, q_over = q_step + a.qs - a.G * a.qh;
    for (int run = rest % a.tiles; run * RUN < end; run += a.tiles) {
        const int run0 = run * RUN, t0 = run0 + w * TOK;
        // ---- the stages of rows that can attend a token of the run, and this work-group's share of them
        const int k_first = max(0, run0 - n);
        const int64_t k_last = run0 < a.sinks ? rows - 1 : min(int64_t(rows) - 1, int64_t(run0) + RUN - 2 - n + a.window);
        const int first = k_first * a.G / SR, last = k_last < k_first ? first : int(((k_last + 1) * a.G + SR - 1) / SR);
        const int per = (last - first + a.shares - 1) / a.shares, s_from = min(first + share * per, last), stages = min(per, last - s_from);
        f32x4 sum[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (stages > 0) {  // (uniform)
            // ---- this lane's rows of a stage: direct load j has row w WR + j RPL + lane / LPR, its log-sum-exps row w WR + lane % WR
            const int r_lane = s_from * SR + w * WR + lane / M::LPR, r_lse = s_from * SR + w * WR + lane % WR;
            const uint16_t* q_at[4];
            int h_at[4], r_at = r_lane, l_at = r_lse, lk_at = r_lse / a.G, lh_at = r_lse % a.G;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r_lane + j * M::RPL;
                h_at[j] = r % a.G;
                q_at[j] = queries + (r / a.G) * a.qs + h_at[j] * a.qh;
            }
            auto issue = [&](int slot) {
                unsigned char* to = smem + slot * 16384 + w * 4096;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // (rows past the last: row 0's, not counted)
                    const int piece = (lane % M::LPR) ^ swizzle<D>((w * WR + j * M::RPL + lane / M::LPR) & 15);
                    const uint16_t* src = (r_at + j * M::RPL < all_rows ? q_at[j] : queries) + piece * 8;
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                                     (__attribute__((address_space(3))) void*)(to + j * 1024), 16, 0, 0);
                    h_at[j] += step_h;
                    const bool over = h_at[j] >= a.G;
                    h_at[j] -= over ? a.G : 0;
                    q_at[j] += over ? q_over : q_step;
                }
                const bool live = l_at < all_rows;
                const uint32_t at = uint32_t(live ? lk_at : 0) * uint32_t(a.H) + uint32_t(live ? lh_at : 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(lse + at),
                                                 (__attribute__((address_space(3))) void*)(smem + NS * 16384 + slot * M::LSE + w * 256), 4, 0, 0);
                r_at += SR;
                l_at += SR;
                lh_at += step_h;
                const bool over = lh_at >= a.G;
                lh_at -= over ? a.G : 0;
                lk_at += step_k + (over ? 1 : 0);
            };
            // ---- the tokens' keys, as A operands
            u32x4 kf[TT][KK];
            uint64_t pages = 0;  // tokens of the wave's that stand in pages
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                const int t = t0 + 16 * i, e = t < end ? uload(trow + (t >> a.lt)) : -1;
                const bool in = uint32_t(e) < uint32_t(a.P);
                pages |= in ? uint64_t(0xFFFF) << (16 * i) : 0;
                // (a tile without a page reads the pool's first rows: in bounds, and selected out)
                const uint16_t* src = a.key + kh * a.kh + (in ? int64_t(e) * a.kp + int64_t(t & ((1 << a.lt) - 1)) * a.kt : 0) + c16 * a.kt + 8 * g;
#pragma unroll
                for (int k = 0; k < KK; ++k) kf[i][k] = *reinterpret_cast<const u32x4*>(src + 32 * k);
            }
            // they have arrived before the first direct load goes out: the compiler waits for all of those before it uses them
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int k = 0; k < KK; ++k) asm volatile("" : "+v"(kf[i][k]));
            __builtin_amdgcn_s_barrier();  // (everyone is done with the ring of the run before)
#pragma unroll
            for (int s = 0; s < NS - 1; ++s)
                if (s < stages) issue(s);
            // Row tiles: from which on and up to which a row of them attends a token of the wave's, and in which every row
            // attends every one.
            const int tile_from = max(0, t0 - n) * a.G / 16;
            const int64_t near_k = int64_t(t0) - n - 1 + a.window, far_k = t0 < a.sinks ? rows - 1 : min(int64_t(rows) - 1, near_k + TOK - 1);
            const int tile_end = pages == 0 || far_k < 0 ? 0 : int(((far_k + 1) * a.G + 15) / 16);
            const int all_k = t0 + TOK - 1 - n;
            const int whole_from = pages != (TOK == 64 ? ~uint64_t(0) : (uint64_t(1) << (TOK & 63)) - 1) ? INT_MAX : all_k <= 0 ? 0 : (all_k * a.G + 15) / 16;
            const int whole_end = t0 + TOK <= a.sinks ? all_rows / 16 : int(max(int64_t(0), min(int64_t(all_rows), (near_k + 1) * a.G)) >> 4);
            const uint32_t q_lane = c16 * M::RB + ((g ^ swizzle<D>(c16)) * 16);
            for (int s = 0; s < stages; ++s) {
                if (s + NS - 2 < stages) wait_vm<LOADS * (NS - 2)>();
                else wait_vm<0>();
                __builtin_amdgcn_s_barrier();  // everyone's share of stage s has landed, everyone is done with stage s - 1
                if (s + NS - 1 < stages) issue((s + NS - 1) % NS);
                const uint32_t at = ring + uint32_t(s % NS) * 16384, lse_at = lse_ring + uint32_t(s % NS) * M::LSE;
#pragma unroll 1
                for (int x = 0; x < SR / 16; ++x) {
                    const int tile = (s_from + s) * (SR / 16) + x;
                    if (tile < tile_from || tile >= tile_end) continue;  // (uniform in the wave)
                    const int row = 16 * x + c16;  // of the stage
                    float base;
                    asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(base) : "v"(lse_at + uint32_t(row / WR * 256 + row % WR * 4)) : "memory");
                    u32x4 qf[KK];
                    read_k<D>(qf, at + q_lane + uint32_t(x) * 16 * M::RB);
                    f32x4 z[TT];
#pragma unroll
                    for (int i = 0; i < TT; ++i) z[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < KK; ++k)
#pragma unroll
                        for (int i = 0; i < TT; ++i) z[i] = E::mfma(kf[i][k], qf[k], z[i]);
                    const float sub = base > -INFINITY ? base * 1.44269504088896340736f : INFINITY;  // (+inf: the row gives nothing)
                    if (tile >= whole_from && tile < whole_end && __builtin_amdgcn_ballot_w64(sub == INFINITY) == 0) {  // (uniform)
#pragma unroll
                        for (int i = 0; i < TT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[i][e] += __builtin_amdgcn_exp2f(fmaf(z[i][e], a.zs, -sub));
                    } else {
                        // the wave's tokens that this row attends: t < lim, of these t < sinks or t >= lim - window
                        const int r = tile * 16 + c16, lim = n + r / a.G + 1 - t0, lo = lim - a.window, f = a.sinks - t0;
                        auto below = [](int m) -> uint64_t { return m <= 0 ? 0 : m >= 64 ? ~uint64_t(0) : (uint64_t(1) << m) - 1; };
                        uint64_t in = sub == INFINITY || r >= all_rows ? 0 : below(lim) & (below(f) | ~below(lo)) & pages;
                        in >>= 4 * g;
#pragma unroll
                        for (int i = 0; i < TT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float p = __builtin_amdgcn_exp2f(fmaf(z[i][e], a.zs, -sub));
                                sum[i][e] += (in >> (16 * i + e)) & 1 ? p : 0.f;
                            }
                    }
                }
            }
        }
        float v[4 * TT];
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = sum[i][e];
        const float mine = row_sums<4 * TT>(v, c16);
        const int t = t0 + 16 * ((c16 % (4 * TT)) >> 2) + 4 * g + (c16 & 3);
        if (c16 >= 4 * TT || t >= end) continue;
        if (a.shares > 1) {
            a.part[((int64_t(share) * a.B + b) * a.Hk + kh) * (int64_t(a.tiles) * RUN) + t] = mine;
        } else {
            const float p = t < n && a.prior ? a.prior[b * a.pb + kh * a.ph + t] : 0.f;
            a.out[b * a.ob + kh * a.oh + t] = p + mine;
        }
    }
}

// The shares' sums joined, in their order.
__global__ __launch_bounds__(256) void attn_mass_join_kernel(MassArgs a, int places) {
    const int blocks = (places + 255) / 256, t = int(blockIdx.x) % blocks * 256 + int(threadIdx.x), kh = int(blockIdx.x) / blocks % a.Hk,
              b = int(blockIdx.x) / blocks / a.Hk;
    const int n = max(0, min(uload(a.length + b), a.W << a.lt));
    const int rows = a.count ? max(0, min(uload(a.count + b), a.S)) : a.S;
    if (t >= min(min(n + rows, a.W << a.lt), a.N)) return;
    float x = 0.f;
    for (int s = 0; s < a.shares; ++s) x += a.part[((int64_t(s) * a.B + b) * a.Hk + kh) * places + t];
    const float p = t < n && a.prior ? a.prior[b * a.pb + kh * a.ph + t] : 0.f;
    a.out[b * a.ob + kh * a.oh + t] = p + x;
}

// ---- launches ---------------------------------------------------------------------------------------------------
constexpr int64_t MOST_GROUPS = 65536;  // work-groups of a launch at most (further runs in a loop)
constexpr int64_t FEW_ROWS = 64;        // query rows of a kv head that a wave goes through by itself
int64_t tiles_of(int64_t tokens, int64_t run, int64_t pairs) {
    const int64_t tiles = (tokens + run - 1) / run;
    return tiles * pairs <= MOST_GROUPS ? tiles : MOST_GROUPS / pairs > 0 ? MOST_GROUPS / pairs : 1;
}
int64_t many_run(int64_t D) { return D == 256 ? Many<256>::RUN : D == 128 ? Many<128>::RUN : Many<64>::RUN; }
// Work-groups that share a run's rows: as many as give every CU three, with four stages at least each (1000 rows over 4000 tokens
// of 8 kv heads, 160 runs: 129 us with one, 94 with two, 70 with three, 61 with five, 67 with six, 63 with eight).
int shares_of(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t tokens) {
    const int64_t runs = B * Hk * ((tokens + many_run(D) - 1) / many_run(D)), stages = (S * (H / Hk) * 2 * D + 16383) / 16384;
    int64_t s = (768 + runs - 1) / runs;
    if (s > 8) s = 8;
    if (s > (stages + 3) / 4) s = (stages + 3) / 4;
    return int(s < 1 ? 1 : s);
}
template <class E, int D>
int launch_many(MassArgs& a, hipStream_t st) {
    using M = Many<D>;
    const int64_t most = int64_t(a.W) << a.lt, tokens = most < a.N ? most : a.N, pairs = int64_t(a.B) * a.Hk;
    static std::atomic<uint64_t> allowed{0};  // (once per device: the call costs about a microsecond)
    int dev = 0;
    MDX_HIP(hipGetDevice(&dev));
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (dev > 63 || !(allowed.load(std::memory_order_relaxed) & bit)) {
        allow_smem(reinterpret_cast<const void*>(&attn_mass_many_kernel<E, D>), M::LDS);
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    a.tiles = int(tiles_of(tokens, M::RUN, pairs));
    hipLaunchKernelGGL((attn_mass_many_kernel<E, D>), dim3(unsigned(a.tiles * pairs * a.shares)), dim3(256), M::LDS, st, a);
    MDX_LAUNCHED();
    if (a.shares > 1) {
        const int places = a.tiles * M::RUN;
        hipLaunchKernelGGL(attn_mass_join_kernel, dim3(unsigned((places + 255) / 256 * pairs)), dim3(256), 0, st, a, places);
        MDX_LAUNCHED();
    }
    return MDX_OK;
}
template <class E, int D, int TT, bool SPLIT, bool PATH>
int launch(MassArgs& a, hipStream_t st) {
    const int64_t most = int64_t(a.W) << a.lt, tokens = most < a.N ? most : a.N, pairs = int64_t(a.B) * a.Hk;
    a.tiles = int(tiles_of(tokens, SPLIT ? 16 * TT : 64 * TT, pairs));
    hipLaunchKernelGGL((attn_mass_kernel<E, D, TT, SPLIT, PATH>), dim3(unsigned(a.tiles * pairs)), dim3(256), 0, st, a);
    MDX_LAUNCHED();
    return MDX_OK;
}
template <class E, int D>
int launch_rows(MassArgs& a, hipStream_t st) {
    constexpr int TT = D == 256 ? 2 : 4;
    if (int64_t(a.S) * a.G <= FEW_ROWS) return a.path ? launch<E, D, TT, false, true>(a, st) : launch<E, D, TT, false, false>(a, st);
    return a.path ? launch<E, D, TT, true, true>(a, st) : launch_many<E, D>(a, st);
}
template <class E>
int launch_any(MassArgs& a, int64_t D, hipStream_t st) {
    return D == 64 ? launch_rows<E, 64>(a, st) : D == 128 ? launch_rows<E, 128>(a, st) : launch_rows<E, 256>(a, st);
}

// Rows of N sums [B, Hk] and their strides.
struct Sums {
    const float* at;
    int64_t sb, sh;
};
// Whether a row of `prior` meets one of `out`, whose rows are apart from one another (views of one buffer may lie in each other's
// gaps): looked up among them row by row, where the ranges meet at all.
bool rows_meet(const Sums& prior, const Sums& out, int64_t B, int64_t Hk, int64_t N) {
    auto bytes = [&](const Sums& x) { return uint64_t((B - 1) * x.sb + (Hk - 1) * x.sh + N) * 4; };
    if (apart(prior.at, bytes(prior), out.at, bytes(out))) return false;
    // out's rows stand at i1 s1 + i2 s2, those of one i1 within s1
    const bool by_head = out.sb < out.sh;
    const int64_t s1 = by_head ? out.sh : out.sb, s2 = by_head ? out.sb : out.sh, n1 = by_head ? Hk : B, n2 = by_head ? B : Hk;
    const int64_t from = (int64_t(reinterpret_cast<uintptr_t>(prior.at)) - int64_t(reinterpret_cast<uintptr_t>(out.at))) / 4;
    // the two rows of stride s that a row at x can meet: those at or ahead of its first place and of its last
    auto near = [](int64_t x, int64_t s, int64_t n) { return s == 0 || x < 0 ? int64_t(0) : x / s < n ? x / s : n - 1; };
    for (int64_t b = 0; b < B; ++b)
        for (int64_t h = 0; h < Hk; ++h) {
            const int64_t x = from + b * prior.sb + h * prior.sh;
            for (const int64_t i1 : {near(x, s1, n1), near(x + N - 1, s1, n1)}) {
                const int64_t y = x - i1 * s1;
                for (const int64_t i2 : {near(y, s2, n2), near(y + N - 1, s2, n2)})
                    if (y - i2 * s2 < N && i2 * s2 - y < N) return true;
            }
        }
    return false;
}

int log2_of(int64_t T) {
    for (int i = 4; i <= 10; ++i)
        if (T == int64_t(1) << i) return i;
    return -1;
}

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_attn_mass_workspace(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t T, int64_t W, int64_t N) {
    if (B < 1 || B > 1024 || S < 1 || S > 65535 || Hk < 1 || Hk > 1024 || H < 1 || H > 65536 || H % Hk != 0 || (D != 64 && D != 128 && D != 256) || T < 16 ||
        T > 1024 || W < 1 || W > (int64_t(1) << 26) || N < 1 || S * (H / Hk) <= FEW_ROWS)
        return 0;
    const int64_t tokens = W * T < N ? W * T : N;
    const int64_t shares = shares_of(B, S, H, Hk, D, tokens);
    return shares == 1 ? 0 : size_t(shares * B * Hk) * size_t(tiles_of(tokens, many_run(D), B * Hk) * many_run(D)) * 4;
}

extern "C" int mdx_attn_mass(const void* q, int64_t q_seq_stride, int64_t q_row_stride, int64_t q_head_stride, const void* key,
                             int64_t k_head_stride, int64_t k_page_stride, int64_t k_row_stride, int32_t dtype, const int32_t* table,
                             int64_t table_stride, const int32_t* length, const float* lse, const float* prior, int64_t prior_seq_stride,
                             int64_t prior_head_stride, const int32_t* count, const int32_t* path, int64_t window, int64_t sinks,
                             float* out, int64_t out_seq_stride, int64_t out_head_stride, int64_t N, int64_t B, int64_t S, int64_t H,
                             int64_t Hk, int64_t D, int64_t P, int64_t T, int64_t W, float scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
    MDX_CHECK(q && key && table && length && lse && out, "null pointer");
    MDX_CHECK(dtype == MDX_DT_BF16 || dtype == MDX_DT_F16, "bf16 or fp16");
    MDX_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
    const int lt = log2_of(T);
    MDX_CHECK(lt >= 0, "page rows: a power of two in 16..1024");
    MDX_CHECK(B >= 1 && B <= 1024 && S >= 1 && S <= 65535 && Hk >= 1 && Hk <= 1024 && H >= 1 && H % Hk == 0 && H <= 65536 && H / Hk <= 128,
              "1..1024 sequences, 1..65535 rows, heads (at most 128 per kv head)");
    MDX_CHECK(P >= 1 && P <= (int64_t(1) << 30) && W >= 1 && (W << lt) < (int64_t(1) << 30) && table_stride >= W &&
                  table_stride <= (int64_t(1) << 26),
              "pages, table [sequences, W], under 2^30 tokens a sequence");
    const int64_t lim = int64_t(1) << 40;
    MDX_CHECK(k_row_stride >= D && k_row_stride <= (int64_t(1) << 24) && k_head_stride >= 0 && k_page_stride >= 0 && k_head_stride < lim &&
                  k_page_stride < lim && q_seq_stride >= 0 && q_row_stride >= 0 && q_head_stride >= 0 && q_seq_stride < lim &&
                  q_row_stride < lim && q_head_stride < lim,
              "strides");
    MDX_CHECK(aligned(q, 16) && aligned(key, 16) && q_seq_stride % 8 == 0 && q_row_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                  k_head_stride % 8 == 0 && k_page_stride % 8 == 0 && k_row_stride % 8 == 0 && aligned(lse, 4) && aligned(out, 4) && aligned(prior, 4),
              "16-byte aligned rows");
    // (rows apart from one another, the sequences' or the kv heads' side by side)
    const int64_t ob = B == 1 ? 0 : out_seq_stride, oh = Hk == 1 ? 0 : out_head_stride;
    MDX_CHECK(N >= 1 && N <= (int64_t(1) << 30) && ob >= 0 && oh >= 0 && ob < lim && oh < lim && (B == 1 || ob >= (Hk - 1) * oh + N || oh >= (B - 1) * ob + N) &&
                  (Hk == 1 || oh >= N) && (B == 1 || ob >= N),
              "sums [sequences, kv heads, places]: apart from one another");
    MDX_CHECK(!prior || (prior_seq_stride >= 0 && prior_head_stride >= 0 && prior_seq_stride < lim && prior_head_stride < lim), "prior strides");
    // (a place is read and written by the same lane)
    const int64_t pb = B == 1 ? 0 : prior_seq_stride, ph = Hk == 1 ? 0 : prior_head_stride;
    MDX_CHECK(prior != out || (pb == ob && ph == oh), "sums in place: prior's strides");
    MDX_CHECK(window >= 1 && window <= (int64_t(1) << 30) && sinks >= 0 && sinks <= (int64_t(1) << 30), "a window of 1..2^30 tokens, 0..2^30 first ones");
    MDX_CHECK(scale > 0.f && scale < INFINITY, "a positive, finite scale");
    MassArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.qb = q_seq_stride, a.qs = q_row_stride, a.qh = q_head_stride;
    a.key = static_cast<const uint16_t*>(key);
    a.kh = k_head_stride, a.kp = k_page_stride, a.kt = k_row_stride;
    a.table = table;
    a.ts = table_stride;
    a.length = length;
    a.lse = lse;
    a.prior = prior;
    a.pb = pb, a.ph = ph;
    a.count = count;
    a.path = path;
    a.out = out;
    a.ob = ob, a.oh = oh;
    a.B = int(B), a.S = int(S), a.H = int(H), a.Hk = int(Hk), a.G = int(H / Hk), a.W = int(W), a.P = int(P), a.lt = lt, a.N = int(N);
    a.window = int(window), a.sinks = int(sinks);
    a.zs = float(double(scale) * 1.4426950408889634);
    const size_t need = path ? 0 : mdx_attn_mass_workspace(B, S, H, Hk, D, T, W, N);  // (rows of a path are not shared out)
    MDX_CHECK(!need || (workspace && aligned(workspace, 16) && workspace_bytes >= need), "workspace: %zu bytes, 16-byte aligned", need);
    // (places are written while others, and queries, are read)
    MDX_CHECK(!prior || prior == out || !rows_meet({prior, pb, ph}, {out, ob, oh}, B, Hk, N), "out: prior itself, or apart from it");
    const uint64_t out_bytes = uint64_t((B - 1) * ob + (Hk - 1) * oh + N) * 4;
    const uint64_t q_bytes = uint64_t((B - 1) * q_seq_stride + (S - 1) * q_row_stride + (H - 1) * q_head_stride + D) * 2;
    MDX_CHECK(apart(out, out_bytes, lse, uint64_t(B * S * H) * 4) && apart(out, out_bytes, q, q_bytes), "out: apart from q and lse");
    a.shares = need ? shares_of(B, S, H, Hk, D, (W << lt) < N ? W << lt : N) : 1;
    a.part = static_cast<float*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == MDX_DT_BF16 ? launch_any<Bf16>(a, D, st) : launch_any<Fp16>(a, D, st);
}
