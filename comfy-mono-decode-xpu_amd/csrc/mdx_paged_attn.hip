// Attention over the paged cache (layout: mdx_pages.hip): single tokens, drafted trees and prompt rows of several
// sequences (mdx_attn_paged), the same over the blocks of a long context that a score selects (mdx_attn_blocks), and within a
// sliding window and a few first tokens, with the rows' log-sum-exps (mdx_attn_window).
//
// Row (b, s, h) attends the committed tokens t < n = length[b] and the rows' own tokens n + j (j < S, their K/V in the
// pages already) that bit j of mask[b][s] admits, or j <= s without masks: softmax(q . k / sqrt(D)) v, 0 where no token
// is admitted. A token in a page that the table does not have is not admitted; what a place holds that a row does not
// admit never reaches it, infinities and NaN included.
//
// Work. A unit is (sequence, kv head, block of query rows); its tokens go in steps of 32 or 64 per token part. The steps of
// all units stand in one line and every work-group takes an equal share of it (one or two work-groups per CU: their rings
// take most of its LDS), so unequal lengths, one long sequence and many short ones keep all CUs busy alike, and the lengths
// are read on the device alone. A share that begins or ends inside a unit leaves a partial (maximum, sum, O in fp32), which
// the second launch joins; a unit inside one share is written at once. Where units are short, or enough of them about equally
// long, a work-group takes a whole one and there is no second launch.
//
// A step of a wave: its 32 tokens' K and V come to LDS by direct loads (1 KiB per wave instruction); S^T = K Q^T with
// A = 16 tokens x 32 dims and B = Q^T in registers (v_mfma_f32_16x16x32), so that the four lanes of a query row hold its
// scores; softmax against an earlier maximum, renewed when a score passes it by a slack; O^T += V^T P^T with A = V^T by transposing LDS reads in the token order the
// S^T accumulators hold, B = P^T from registers. A wave holds up to four tiles of 16 query rows and reads each K and V
// operand once for all of them. Sums, maxima and O in fp32; P is rounded to the cache's type for the product (half a
// step of each weight; the normaliser sums the rounded weights, so that equal values come out unchanged; a log-sum-exp is that of
// the weights as they were).
//
// What bounds it. Few rows: the cache's bytes, where there are many (64 single tokens over 262 thousand: 193 us, 5.6 TB/s),
// else the latency of one work-group's chain of queries, pages, first stage, products, meeting and join (one token of a
// short sequence: 6 us in a whole unit). Many rows: the matrix units' and the softmax's instructions in turn, with two waves per
// SIMD to overlap them (2048 rows over 30000 tokens: 1027 us, 1.0 PFLOP/s of the 1.2 that a large matrix product reaches;
// 64 tokens a stage instead of 32: 128 -> 99 us for 2048 rows over 1000).
//
// Reference: none for the pages; the rows' contract is csrc/attn_dpas.sycl:269-342's.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <atomic>

#include "mdx_lds.hpp"

namespace mdx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// The two element types: their MFMA, and P's rounding. fp16 holds weights down to 2^-14 at full precision only: P is
// scaled by 2^14 there (exact; numerator and normaliser alike), so weights down to 2^-28 of the largest keep theirs.
// SLACK: how far (log2) scores may pass the row's reference before the sums are brought to a new one; fp16 holds weights up
// to 2^(14 + SLACK).
struct Bf16 {
    static constexpr float SHIFT = 0.f, SLACK = 8.f;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(mdx_f32x2{a, b}, mdx_bf16x2));
    }
    static __device__ __forceinline__ float add_pair(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(mdx_bf16x2, p), mdx_bf16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
    }
    static __device__ __forceinline__ float to_f32(uint16_t x) { return bf2f(x); }
    static constexpr uint32_t EXP = 0x7F807F80u, ONE = 0x00800080u;  // two elements' exponents, one step of them
};
struct Fp16 {
    static constexpr float SHIFT = 14.f, SLACK = 1.5f;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(mdx_f32x2{a, b}, f16x2));
    }
    static __device__ __forceinline__ float add_pair(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
    }
    static __device__ __forceinline__ float to_f32(uint16_t x) { return fp16_to_f32(x); }
    static constexpr uint32_t EXP = 0x7C007C00u, ONE = 0x04000400u;
};

struct PagedArgs {
    const uint16_t* q;  // [B, S, H, D], strides qb, qs, qh
    int64_t qb, qs, qh;
    const uint16_t* key;  // [Hk, P, T, D], strides kh, kp, kt
    int64_t kh, kp, kt;
    const uint16_t* value;
    int64_t vh, vp, vt;
    const int32_t* table;  // [B, W], row stride ts
    int64_t ts;
    const int32_t* length;  // [B]
    const int64_t* mask;    // [B, S] or null (a chain)
    uint16_t* out;          // [B, S, H, D]
    // selected blocks (mdx_attn_blocks): page indices of the table and pages of the pool, [B, S, Hk, most]
    int32_t* sel;
    int32_t* page;
    int most, sink, local;
    const uint16_t* ksum;  // [Hk, P, D], strides sh, sp
    int64_t sh, sp;
    uint64_t* keys;  // [B, S, Hk, W]
    int4* info;      // the units left open to join: (unit, first share, shares), by unit (where they are few) or by share
    int by_unit;
    float* part;     // [2 work-groups][rows][D + 2]: O, maximum, sum
    int B, S, H, Hk, G, W, P, lt;
    int units;  // units of a sequence and kv head: blocks of spb rows s (1 with a selection each)
    int spb;    // a unit's query rows: s from u spb, each with the kv head's G heads
    int whole;  // every work-group takes one whole unit (no join)
    float zs;   // scale * log2(e)
    // a row's first `first` and last `window` tokens (mdx_attn_window), and its log-sum-exp [B, S, H]
    int first, window;
    float* lse;
};

// What a row's tokens are: all that are admitted, those of selected blocks (mdx_attn_blocks), or its first and last ones
// (mdx_attn_window).
enum class Kind { ALL, SEL, WIN };
// fp32 numbers of a partial beside O: maximum, sum (windows: and the sum of the weights before their rounding)
constexpr int extra_of(Kind k) { return k == Kind::WIN ? 3 : 2; }

constexpr int MAX_SEQS = 1024;
constexpr int STEP = 32;
// References (log2 units) past which scores are taken less the reference in score units first. A weight's exponent is
// score * zs - reference * zs, the first product unrounded, the second one fp32 number: its rounding (2^-9 up to here) is a
// factor that numerator and normaliser share. Further out it grows past what the weights' type holds (fp16 from 2^26 on, bf16
// from 2^32: NaN for finite inputs).
constexpr float FAR_REF = 65536.f;
constexpr int CUS = 256;
// Steps of all units together, with their fixed cost: positions are 32-bit numbers, and the last shares' ends pass the line's by
// up to one step for each of 2 CUS shares.
constexpr int64_t MAX_LINE = (int64_t(1) << 31) - 4 * CUS;
constexpr int RING_BYTES = 128 * 1024;  // of a CU's work-groups together
// 128-token steps of a call at most, for the forms that go by latency (below: launch_rows)
constexpr int64_t FEW_STEPS = 2048;
// The forms go by what the table could hold, the lengths being on the device alone; a caller with a bound on them passes a table
// of fewer columns (all rules measured with tables as wide as the lengths).
// Tokens a unit can have at most, for one work-group per unit: 8 units of one token over 500: 9.4 us a call, 12.6 in shares
// with their join; of 16 rows over 500: 15.5 and 13.9, 128 of them 16.5 and 25.3. Twice as many where the units fill half of
// the CUs and no more than all (128 units of one token over 1000: 15.7 and 20.2, of 16 rows 23.0 and 29.3; 8 units of one
// token over 1000: 13.2 and 11.7).
constexpr int64_t WHOLE_TOKENS = 640;
constexpr int64_t EVEN_TOKENS = 4096;  // and where there are as many row blocks as work-groups

// LDS layout of a 32-token stage, K and V alike: the tokens' rows of 2 D bytes one after the other, as they stand in a page,
// so that a direct load's KiB is one KiB of the page (64-byte pieces of 16 tokens per load took 2 % longer, 200 us against 196
// for 64 single-token sequences of 262 thousand tokens in all). Within a row the 16-byte pieces are exchanged by
// an exclusive or with the token (swizzle), which the loads' source addresses follow, so that
//   K: lane (token c16 of the half, k-group g) reads piece 4 kk + g, 16 tokens of one piece meeting all banks once;
//   V: the transposing reads (lane s of group g points at token 4 g + s / 4 of the half, dims 16 dt + 4 (s % 4) .. + 3, and
//      receives dim c16 of tokens 4 g .. 4 g + 3) meet every bank alike;
// both from one lane address: piece bits above the lane's own enter by an exclusive or with a constant.
// The reads are inline asm that ends with its wait: the builtins would wait for every direct load in flight.
// both halves at once
template <int D>
__device__ __forceinline__ void read_k2(u32x4 (&kf)[2][D / 32], uint32_t at) {
    if constexpr (D == 128) {
        asm volatile(
            "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
            "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\t"
            "ds_read_b128 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(kf[0][0]), "=&v"(kf[0][1]), "=&v"(kf[0][2]), "=&v"(kf[0][3]), "=&v"(kf[1][0]), "=&v"(kf[1][1]),
              "=&v"(kf[1][2]), "=&v"(kf[1][3])
            : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
            : "memory");
    } else {
        read_k<D>(kf[0], at);
        read_k<D>(kf[1], at + 16 * 2 * D);
    }
}
// V^T of dim tiles 8 X .. 8 X + 7 (D = 64: the four there are): va tokens of half 0, vb of half 1
template <int D, int X>
__device__ __forceinline__ void read_v(u32x2 (&va)[D == 64 ? 4 : 8], u32x2 (&vb)[D == 64 ? 4 : 8], uint32_t at) {
    if constexpr (D == 64) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %2, %10\n\t"
            "ds_read_b64_tr_b16 %3, %11\n\tds_read_b64_tr_b16 %4, %8 offset:2048\n\tds_read_b64_tr_b16 %5, %9 offset:2048\n\t"
            "ds_read_b64_tr_b16 %6, %10 offset:2048\n\tds_read_b64_tr_b16 %7, %11 offset:2048\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(va[0]), "=&v"(va[1]), "=&v"(va[2]), "=&v"(va[3]), "=&v"(vb[0]), "=&v"(vb[1]), "=&v"(vb[2]), "=&v"(vb[3])
            : "v"(at), "v"(at ^ 32), "v"(at ^ 64), "v"(at ^ 96)
            : "memory");
    } else {
        static_assert(D == 128 || D == 256, "");
        asm volatile(
            "ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %1, %17 offset:%24\n\t"
            "ds_read_b64_tr_b16 %2, %18 offset:%24\n\tds_read_b64_tr_b16 %3, %19 offset:%24\n\t"
            "ds_read_b64_tr_b16 %4, %20 offset:%24\n\tds_read_b64_tr_b16 %5, %21 offset:%24\n\t"
            "ds_read_b64_tr_b16 %6, %22 offset:%24\n\tds_read_b64_tr_b16 %7, %23 offset:%24\n\t"
            "ds_read_b64_tr_b16 %8, %16 offset:%25\n\tds_read_b64_tr_b16 %9, %17 offset:%25\n\t"
            "ds_read_b64_tr_b16 %10, %18 offset:%25\n\tds_read_b64_tr_b16 %11, %19 offset:%25\n\t"
            "ds_read_b64_tr_b16 %12, %20 offset:%25\n\tds_read_b64_tr_b16 %13, %21 offset:%25\n\t"
            "ds_read_b64_tr_b16 %14, %22 offset:%25\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(va[0]), "=&v"(va[1]), "=&v"(va[2]), "=&v"(va[3]), "=&v"(va[4]), "=&v"(va[5]), "=&v"(va[6]), "=&v"(va[7]),
              "=&v"(vb[0]), "=&v"(vb[1]), "=&v"(vb[2]), "=&v"(vb[3]), "=&v"(vb[4]), "=&v"(vb[5]), "=&v"(vb[6]), "=&v"(vb[7])
            : "v"(at), "v"(at ^ 32), "v"(at ^ 64), "v"(at ^ 96), "v"(at ^ 128), "v"(at ^ 160), "v"(at ^ 192), "v"(at ^ 224),
              "n"(X * 256), "n"(X * 256 + 16 * 2 * D)
            : "memory");
    }
}

typedef __attribute__((address_space(4))) const int32_t* const_i32p;
__device__ __forceinline__ int uload(const int32_t* p) { return *(const_i32p)(p); }  // (a scalar load: uniform addresses)

// the largest of three (a NaN counts as the smallest; fmaxf would first make every operand a quiet one)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The tokens a unit's steps run over, as virtual tokens v: the first `nsel` of them are selected blocks' (Kind::SEL) or the
// sequence's first ones (Kind::WIN), the others are tokens tail + (v - nsel) in a row. Kind::ALL: [0, n + own rows).
struct Span {
    int n;      // committed tokens
    int tree0;  // virtual token of own row 0 (of a window that begins among the rows' own tokens: negative)
    int nsel;   // tokens of selected blocks, or first ones in whole stages (0: none)
    int tail;   // token at which the tail starts
};
constexpr int WIN_STEP = 64;  // a window's parts begin at multiples of the longest stage
// own tokens that unit u attends at most (a chain's unit ends with its last row's)
__device__ __forceinline__ int own_of(const PagedArgs& a, int u) { return a.mask ? a.S : min(a.S, (u + 1) * a.spb); }
template <Kind KIND>
__device__ __forceinline__ Span span_of(const PagedArgs& a, int n, int u) {
    n = n < 0 ? 0 : (n > (a.W << a.lt) ? a.W << a.lt : n);
    if constexpr (KIND == Kind::ALL) return {n, n, 0, 0};
    if constexpr (KIND == Kind::WIN) {
        // the window of the unit's first row (under a mask: of a row without own tokens), and the first tokens, as one part
        // where they meet
        const int lo = n + (a.mask ? 0 : u * a.spb + 1) - a.window, tail = lo > 0 ? lo & ~(WIN_STEP - 1) : 0;
        const int nsel = (min(a.first, n + own_of(a, u)) + WIN_STEP - 1) & ~(WIN_STEP - 1);
        if (tail <= nsel) return {n, n, 0, 0};
        return {n, nsel + n - tail, nsel, tail};
    }
    const int c = n >> a.lt, k = c < a.most ? c : a.most;
    return {n, (k << a.lt) + (n - (c << a.lt)), k << a.lt, c << a.lt};
}
// A row's own tokens under a mask (bits) that a window leaves: of all its tokens, the n committed and these in order, the first
// `first` and the last `window`.
__device__ __forceinline__ uint64_t own_in_window(const PagedArgs& a, uint64_t bits, int n) {
    uint64_t left = bits;
    for (int i = 0, gone = __popcll(bits) - a.window; i < gone; ++i) {
        const uint64_t low = left & (0 - left);
        left ^= low;
        if (n + i >= a.first) bits ^= low;
    }
    return bits;
}
__device__ __forceinline__ int steps_of(const PagedArgs& a, const Span& s, int u, int tokens_per_step) {
    return (s.tree0 + own_of(a, u) + tokens_per_step - 1) / tokens_per_step;
}

// log(sum of exp(scores)) of weights that are taken against M (log2 units), times 2^SHIFT; -inf for none
template <class E>
__device__ __forceinline__ float log_sum(float M, float sum) {
    return sum == 0.f ? -INFINITY : (M + (__builtin_amdgcn_logf(sum) - E::SHIFT)) * 0.69314718055994530942f;
}

// One work-group: RTW waves of row tiles (TPW tiles of 16 query rows each) times P token parts.
// (WPC of them share a CU: waves that meet at a barrier are then not all of the CU's)
template <int D, int TPW, int RTW, int P, int WPC, int SUB>
struct Geometry {
    static constexpr int NT = 64 * RTW * P;
    static constexpr int RPW = 16 * TPW * RTW;
    static constexpr int STAGE = STEP * SUB * 2 * D;              // bytes of K (or V) per stage of SUB 32-token pieces
    static constexpr int RING = RING_BYTES / WPC;
    static constexpr int NS = RING / (2 * STAGE * P);             // ring stages per part
    static constexpr int PER = STAGE / 1024 / RTW;                // direct loads per wave, stage and matrix
    // What a unit costs beside its steps (its queries, the ring's first stage, the meeting of its parts), in steps: without
    // it the share that takes the shortest units ends last. 16 prompts of 128 rows over 0 to 6000 tokens: 408 us a call with
    // 0, 167 with 6, 160 with 5; 64 trees of 16 rows over at most 900: 104 with 0, 59 with 4; 48 over at most 8192 at head_dim
    // 64: 119 with 4, 112 with 5; trees of 8 rows: 159 with 4, 156 with 3; 16 single tokens over at most 8192: 48 with 0, 44
    // with 2; of 64 sequences' selections, one with 256 blocks and the others with 4: 199 with 0, 223 with 2.
    static constexpr int FIXED = RPW == 16 ? 2 : RPW == 32 ? 3 : 5;
    static_assert(NS >= 1 && (NS & (NS - 1)) == 0 && PER >= 1 && (RTW == 1 ? SUB == 1 : NS >= 2) && (SUB == 1 || D != 256), "ring geometry");
};

template <class E, int D, int TPW, int RTW, int P, int WPC, int SUB, Kind KIND>
__global__ __launch_bounds__(64 * RTW * P, RTW * P * WPC / 4) void paged_attn_kernel(PagedArgs a) {
    constexpr bool SEL = KIND == Kind::SEL, WIN = KIND == Kind::WIN;
    using Geo = Geometry<D, TPW, RTW, P, WPC, SUB>;
    constexpr int NT = Geo::NT, RPW = Geo::RPW, STAGE = Geo::STAGE, NS = Geo::NS, PER = Geo::PER;
    constexpr int KK = D / 32, DT = D / 16, ST = STEP * SUB, TOK = ST * P;
    extern __shared__ __align__(256) unsigned char smem[];  // (the reads' exclusive ors need rows aligned to 256 bytes)
    __shared__ int sh_sum[NT / 64], sh_at[4];
    __shared__ int odd[2];  // the first and the last stage of the unit that left values out which a row attends (none: -1 last)
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    const int rw = w % RTW, part = w / RTW;
    // Work-groups go to the 8 XCDs in turn: each XCD takes neighbouring shares, so that the row blocks of a kv head, which
    // read the same K and V, find them in one L2 (a prompt's 2048 rows in shares: 144 us, and 164 with the shares in turn; both
    // before the steps of 64 tokens).
    const int share = a.whole ? int(blockIdx.x) : int(blockIdx.x) % 8 * (CUS * WPC / 8) + int(blockIdx.x) / 8;

    int begin, end, quota, b, in_b, kh = 0, u = 0;
    Span sp;
    auto next_unit = [&]() {
        if (++u == a.units) {
            u = 0;
            if (++kh == a.Hk) {
                kh = 0;
                ++b;
                sp = span_of<KIND>(a, uload(a.length + b), u);
            }
        }
        if constexpr (WIN) sp = span_of<KIND>(a, sp.n, u);
    };

    // ---- this work-group's share of the line of steps: [begin, end), and the sequence it begins in
    if (a.whole) {  // unit (b, kh, u) of the grid
        // kv heads in turn (neighbouring work-groups go to different XCDs), a chain's blocks with the most tokens first; every
        // second round of the CUs the other way, so that a CU's work-groups have about as much to do together.
        kh = int(blockIdx.x) % a.Hk;
        const int rest = int(blockIdx.x) / a.Hk, all = a.B * a.units, turn = CUS / a.Hk > 0 ? CUS / a.Hk : 1, q = rest / turn;
        const int rank = (q & 1) && (q + 1) * turn <= all ? 2 * q * turn + turn - 1 - rest : rest;
        b = rank % a.B;
        u = a.units - 1 - rank / a.B;
        sp = span_of<KIND>(a, uload(a.length + b), u);
        begin = in_b = 0;
        end = quota = steps_of(a, sp, u, TOK);
        if (tid == 0) odd[0] = INT_MAX, odd[1] = -1;
    } else {
        // The units in the line's order (sequence, kv head, block), a run of neighbouring ones per thread (where a kv head
        // is one unit, its sequence's kv heads together); the threads' sums, and the unit that the share begins in.
        const int per_kh = a.units == 1 ? a.Hk : 1, n_items = a.units == 1 ? a.B : a.B * a.Hk * a.units;
        const int each = (n_items + NT - 1) / NT, i0 = min(tid * each, n_items), i1 = min(i0 + each, n_items);
        const int per_b = a.units == 1 ? 1 : a.Hk * a.units;
        // (f(item's sequence, its unit, its steps) over this thread's items)
        auto walk = [&](auto f) {
            int bb = i0 / per_b, rest = i0 % per_b, uu = rest % a.units;
            for (int i = i0; i < i1; ++i) {
                f(bb, rest, steps_of(a, span_of<KIND>(a, a.length[bb], uu), uu, TOK) + Geo::FIXED);
                if (++uu == a.units) uu = 0;
                if (++rest == per_b) {
                    rest = 0;
                    ++bb;
                }
            }
        };
        int sum = 0;
        walk([&](int, int, int n) { sum += n * per_kh; });
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(incl, d, 64);
            if (lane >= d) incl += x;
        }
        if (lane == 63) sh_sum[w] = incl;
        __syncthreads();
        int total = 0, before = incl - sum;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            const int x = sh_sum[i];
            before += i < w ? x : 0;
            total += x;
        }
        quota = (total + int(gridDim.x) - 1) / int(gridDim.x);
        begin = share * quota;
        end = min(total, begin + quota);
        if (begin >= before && begin < before + sum)
            walk([&](int bb, int rest, int n) {
                const int in = begin - before;
                if (in >= 0 && in < n * per_kh) {
                    sh_at[0] = bb;
                    sh_at[1] = a.units == 1 ? in / n : rest / a.units;
                    sh_at[2] = a.units == 1 ? 0 : rest % a.units;
                    sh_at[3] = in % n;
                }
                before += n * per_kh;
            });
        if (tid == 0) {
            if (!a.by_unit) a.info[share] = make_int4(0, 0, 0, 0);
            odd[0] = INT_MAX, odd[1] = -1;
        }
        if (begin >= end) return;  // (uniform)
        __syncthreads();
        begin = __builtin_amdgcn_readfirstlane(begin);
        end = __builtin_amdgcn_readfirstlane(end);
        quota = __builtin_amdgcn_readfirstlane(quota);
        b = __builtin_amdgcn_readfirstlane(sh_at[0]);
        kh = __builtin_amdgcn_readfirstlane(sh_at[1]);
        u = __builtin_amdgcn_readfirstlane(sh_at[2]);
        in_b = __builtin_amdgcn_readfirstlane(sh_at[3]);
        sp = span_of<KIND>(a, uload(a.length + b), u);
        const int past = in_b - steps_of(a, sp, u, TOK);
        if (past >= 0) {  // (behind the unit's last step: the next unit)
            begin += Geo::FIXED - past;
            if (begin >= end) return;
            in_b = 0;
            next_unit();
        }
    }
    __syncthreads();  // (odd)
    int at = begin, step0 = in_b;  // line position, and the unit's step there

    unsigned char* ring = smem + part * NS * 2 * STAGE;
    const uint32_t ring_lds = lds_addr(ring);
    constexpr int RB = 2 * D, LPR = RB / 16, TPL = 64 / LPR;  // bytes and pieces of a token's row, tokens per direct load
    const uint32_t k_lane = c16 * RB + ((g ^ swizzle<D>(c16)) * 16);
    const int v_tok = 4 * g + (c16 >> 2);
    const uint32_t v_lane = v_tok * RB + ((((c16 & 3) >> 1) ^ swizzle<D>(v_tok)) * 16) + (c16 & 1) * 8;
    // The lane's place within a direct load: token lane / LPR, piece lane % LPR as exchanged; load i of a matrix covers the
    // tokens from TPL i, whose swizzle enters by an exclusive or (swizzle(TPL i + x) = swizzle(TPL i) ^ swizzle(x)).
    const uint32_t piece = ((lane % LPR) ^ swizzle<D>(lane / LPR)) * 16;
    const uint64_t page_k = uint64_t(a.kp) * 2, page_v = uint64_t(a.vp) * 2;  // (bytes)
    const uint32_t row_k = uint32_t(a.kt) * 2, row_v = uint32_t(a.vt) * 2;
    const uint32_t k_row = (lane / LPR) * uint32_t(a.kt) * 2, v_row = (lane / LPR) * uint32_t(a.vt) * 2;

    while (true) {
        const int n_unit = steps_of(a, sp, u, TOK);
        const int nst = min(n_unit - step0, end - at);  // steps of this unit in the share
        const int t_end = sp.tree0 + own_of(a, u);
        const int s_first = u * a.spb, rows = min(a.spb, a.S - s_first) * a.G;  // query rows of the unit

        // tokens that every row of the wave admits (a chain's first row in the wave its own too)
        const int t_all = sp.tree0 + (a.mask ? 0 : min(a.S, s_first + rw * TPW * 16 / a.G + 1));
        const int t_none = a.mask ? t_end : min(t_end, sp.tree0 + s_first + ((rw + 1) * TPW * 16 - 1) / a.G + 1);  // from here none
        // windows: tokens from which the wave's first and its last row attend (under masks: rows of no own tokens, of all)
        const int lo_first = WIN ? sp.n - a.window + (a.mask ? 0 : s_first + rw * TPW * 16 / a.G + 1) : 0;
        const int lo_last = WIN ? sp.n - a.window + (a.mask ? a.S : min(a.S, s_first + ((rw + 1) * TPW * 16 - 1) / a.G + 1)) : 0;

        // ---- the pages of a stage (scalar loads ahead of their use), and its direct loads
        const unsigned char* kbase = reinterpret_cast<const unsigned char*>(a.key + kh * a.kh);
        const unsigned char* vbase = reinterpret_cast<const unsigned char*>(a.value + kh * a.vh);
        const int32_t* row = a.table + b * a.ts;
        const int32_t* picked = SEL ? a.page + ((int64_t(b) * a.S + u) * a.Hk + kh) * a.most : nullptr;
        constexpr int QT = 2 * SUB;  // 16-token pieces of a stage, each of one page
        struct Pages {
            int e[QT];
        };
        const bool one_page = a.lt >= (SUB == 1 ? 5 : 6);  // (a stage's tokens stand in one page)
        auto entry = [&](int v) {
            if (v >= t_end) return -1;
            if (SEL && v < sp.nsel) return uload(picked + (v >> a.lt));
            const int j = (SEL || (WIN && v >= sp.nsel) ? sp.tail + (v - sp.nsel) : v) >> a.lt;
            return j < a.W ? uload(row + j) : -1;
        };
        auto entries = [&](int s) {
            const int v0 = (step0 + s) * TOK + part * ST;
            Pages x;
            x.e[0] = entry(v0);
#pragma unroll
            for (int h = 1; h < QT; ++h) x.e[h] = one_page ? 0 : entry(v0 + 16 * h);  // (one page: unused; a copy would wait here)
            return x;
        };
        uint32_t hist = 0;  // QT bits per stage issued: its 16-token pieces stand in pages
        // A wave's loads of a stage lie in one piece where several waves share them: only that piece's address is formed.
        constexpr int HALF = 16 / TPL;  // loads of a piece
        constexpr int HW = PER <= HALF ? 1 : 2;
        static_assert(HW == 1 || SUB == 1, "");
        const int h_own = HW == 1 ? rw * PER / HALF : 0;  // (the wave's piece)
        const unsigned char *kp_[HW], *vp_[HW];
        auto place = [&](int s, Pages x) {
            const int v0 = (step0 + s) * TOK + part * ST;
            const uint32_t r0 = uint32_t(SEL && v0 >= sp.nsel ? v0 - sp.nsel : WIN && v0 >= sp.nsel ? v0 - sp.nsel + sp.tail : v0);
            const bool in0 = uint32_t(x.e[0]) < uint32_t(a.P);
            uint32_t ok = in0 ? (1u << QT) - 1u : 0u;
            int e_own = x.e[0];
            if (!one_page) {
                ok = in0 ? 1u : 0u;
#pragma unroll
                for (int h = 1; h < QT; ++h) {
                    ok |= uint32_t(x.e[h]) < uint32_t(a.P) ? 1u << h : 0u;
                    e_own = h_own == h ? x.e[h] : e_own;
                }
            }
            hist = (hist << QT) | ok;
#pragma unroll
            for (int i = 0; i < HW; ++i) {
                if (i == 1 && one_page) {
                    kp_[HW - 1] = kp_[0] + 16 * row_k;
                    vp_[HW - 1] = vp_[0] + 16 * row_v;
                    break;
                }
                // (a piece without a page reads the pool's first rows: in bounds, and masked)
                const int h = HW == 1 ? h_own : i, own = HW == 1 ? e_own : x.e[i];
                const bool in = uint32_t(own) < uint32_t(a.P);
                const uint32_t e = in ? uint32_t(own) : 0u;
                const uint32_t r = in ? (r0 + 16 * h) & ((1u << a.lt) - 1u) : 0u;
                kp_[i] = kbase + (uint64_t(e) * page_k + uint64_t(r) * row_k);
                vp_[i] = vbase + (uint64_t(e) * page_v + uint64_t(r) * row_v);
            }
        };
        auto load = [&](const unsigned char* const (&from)[HW], uint32_t lane_row, uint32_t stride, unsigned char* dst) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = HW == 1 ? rw * PER % HALF + j : j;  // load of its half, or of the stage: tokens TPL i ..
                const unsigned char* src = from[HW == 1 ? 0 : j / HALF] +
                                           (lane_row + uint32_t((i % HALF) * TPL) * stride + (piece ^ uint32_t(swizzle<D>(TPL * (i % HALF)) * 16)));
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                                 (__attribute__((address_space(3))) void*)(dst + (rw * PER + j) * 1024), 16, 0, 0);
            }
        };
        auto issue_k = [&](int s) { load(kp_, k_row, row_k, ring + (s & (NS - 1)) * 2 * STAGE); };
        auto issue_v = [&](int s) { load(vp_, v_row, row_v, ring + (s & (NS - 1)) * 2 * STAGE + STAGE); };
        // A wave with a ring of its own (RTW == 1) fills the whole ring ahead, refills K's slot once it has read K and V's
        // once it has read V, and meets no barrier. Waves that share a ring fill NS - 1 stages ahead and refill the slot of
        // the stage before at the top of a stage, behind the one barrier.
        constexpr int AHEAD = RTW == 1 ? NS : NS - 1;
        Pages first_e[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) first_e[s] = entries(s);

        // ---- query rows and what they admit
        u32x4 qf[TPW][KK];
        uint64_t bits[TPW];
        int lim[TPW], lo[TPW];  // a chain's row; the first token of its window
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            const int r = (rw * TPW + t) * 16 + c16, rr = r < rows ? r : 0;
            const int s = s_first + rr / a.G, h = kh * a.G + rr % a.G;
            const uint16_t* src = a.q + b * a.qb + s * a.qs + h * a.qh + 8 * g;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) qf[t][kk] = *reinterpret_cast<const u32x4*>(src + 32 * kk);
            bits[t] = a.mask ? uint64_t(a.mask[int64_t(b) * a.S + s]) : 0;
            if (a.S < 64) bits[t] &= (uint64_t(1) << a.S) - 1;
            lim[t] = s;
            lo[t] = 0;
        }
        // they have arrived before the first direct load goes out: the compiler waits for all of those before it uses a
        // register that a load among them wrote
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+v"(qf[t][kk]));
            asm volatile("" : "+v"(bits[t]));
            if constexpr (WIN) {
                lo[t] = sp.n - a.window + (a.mask ? __popcll(bits[t]) : lim[t] + 1);
                if (a.mask) bits[t] = own_in_window(a, bits[t], sp.n);
            }
        }

        f32x4 acc[TPW][DT];
        // per row: the score up to which its reference serves (-inf: none yet; the lowest number: past FAR_REF, every stage
        // looks), the reference, an earlier maximal score (0 as long as nothing is admitted, so that -inf - -inf never forms), the
        // sum of weights
        float m_lim[TPW], m_ref[TPW], l[TPW];
        float lx[TPW];  // windows: the sum of the weights before their rounding (the log-sum-exp's)
        const float slack = E::SLACK / a.zs;
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            m_lim[t] = -INFINITY;
            m_ref[t] = 0.f;
            l[t] = lx[t] = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (s < nst) {
                place(s, first_e[s]);
                issue_k(s);
                issue_v(s);
            }
        Pages next_e = entries(AHEAD);  // of the stage issued next
        for (int s = 0; s < nst; ++s) {
            const uint32_t slot = ring_lds + (s & (NS - 1)) * 2 * STAGE;
            // (stages issued when stage s is read: AHEAD more, as far as there are any)
            const int behind = min(nst - s, AHEAD) - 1;
            const uint32_t ok = (hist >> (QT * behind)) & ((1u << QT) - 1u);
            const bool more = s + AHEAD < nst;
            if constexpr (RTW == 1) {
                if (s + AHEAD - 1 < nst) wait_vm<PER * (2 * NS - 1)>();
                else wait_vm<0>();
            } else {
                if (s + AHEAD - 1 < nst) wait_vm<2 * PER * (AHEAD - 1)>();
                else wait_vm<0>();
                __builtin_amdgcn_s_barrier();  // everyone's share of stage s has landed, everyone is done with stage s - 1
                if (more) {
                    place(s + AHEAD, next_e);
                    issue_k(s + AHEAD);
                    issue_v(s + AHEAD);
                    next_e = entries(s + AHEAD + 1);
                }
            }
            const int v0 = (step0 + s) * TOK + part * ST;
            if (RTW > 1 && v0 >= t_none) continue;  // (uniform in the wave: only its loads and the barriers are left)
            // windows: the token of v0, the virtual one of own row 0 in this part of the span
            const int r0 = WIN && v0 >= sp.nsel ? v0 - sp.nsel + sp.tail : v0, tree0 = WIN && v0 < sp.nsel ? sp.n : sp.tree0;
            if (WIN && RTW > 1 && r0 >= a.first && r0 + ST <= lo_first && r0 + ST <= sp.n + (a.mask ? 0 : a.S)) continue;
            f32x4 st[SUB][TPW][2];
            auto scores = [&](const u32x4 (&k)[KK], int x, int h) {
#pragma unroll
                for (int t = 0; t < TPW; ++t) {
                    st[x][t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk) st[x][t][h] = E::mfma(k[kk], qf[t][kk], st[x][t][h]);
                }
            };
            auto refill_k = [&]() {
                if (RTW == 1 && more) {
                    place(s + AHEAD, next_e);
                    issue_k(s + AHEAD);
                }
            };
            if constexpr (D == 256) {  // (half by half: the operands of one half are 32 registers)
                u32x4 kf[KK];
                read_k<D>(kf, slot + k_lane);
                scores(kf, 0, 0);
                read_k<D>(kf, slot + k_lane + 16 * RB);
                refill_k();
                scores(kf, 0, 1);
            } else {
                u32x4 kf[SUB][2][KK];
#pragma unroll
                for (int x = 0; x < SUB; ++x) {
                    read_k2<D>(kf[x], slot + k_lane + x * STEP * RB);
                    if (x == SUB - 1) refill_k();
                    scores(kf[x][0], x, 0);
                    scores(kf[x][1], x, 1);
                }
            }

            // (uniform in the wave) every row admits every token
            const bool whole = ok == (1u << QT) - 1u && v0 + ST <= (WIN ? t_all - sp.tree0 + tree0 : t_all) &&
                               (!WIN || r0 + ST <= a.first || r0 >= lo_last);
            // which of the 32 tokens from r on are among the first, or from `from` on (Kind::WIN)
            auto in_window = [&](int r, int from) -> uint32_t {
                const int f = a.first - r, k = from - r;
                return (f >= 32 ? ~0u : (f > 0 ? (1u << f) - 1u : 0u)) | (k <= 0 ? ~0u : (k < 32 ? ~0u << k : 0u));
            };
            // tile t's weights of the stage, as the B operands of O^T += V^T P^T
            struct Weights {
                u32x4 p[SUB];
            };
            auto weights = [&](int t) -> Weights {
                Weights r;
                if (!whole) {
                    bool any = false;
#pragma unroll
                    for (int x = 0; x < SUB; ++x) {
                        int p = (WIN ? tree0 : sp.tree0) - v0 - STEP * x;  // tokens of the prefix in the piece
                        asm volatile("" : "+s"(p));        // (none of this ahead of the branch)
                        const uint32_t near = WIN ? in_window(r0 + STEP * x, lo[t]) : ~0u;
                        uint32_t in;
                        if (a.mask) {
                            const uint64_t own_bits = p >= 32 ? 0 : (p >= 0 ? bits[t] << p : (-p < 64 ? bits[t] >> -p : 0));
                            in = ((p >= 32 ? ~0u : (p > 0 ? (1u << p) - 1u : 0u)) & near) | uint32_t(own_bits);
                        } else {
                            const int nv = p + lim[t] + 1;
                            in = (nv >= 32 ? ~0u : (nv > 0 ? (1u << nv) - 1u : 0u)) & near;
                        }
                        const uint32_t here = ok >> (2 * x);
                        in &= ((here & 1u) ? 0x0000FFFFu : 0u) | ((here & 2u) ? 0xFFFF0000u : 0u);
                        any = any || __builtin_amdgcn_ballot_w64(in != 0u) != 0;
                        const uint32_t lb = in >> (4 * g);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (!((lb >> (16 * h + i)) & 1u)) st[x][t][h][i] = -INFINITY;
                    }
                    if (!any) {  // (uniform: nothing for this tile)
#pragma unroll
                        for (int x = 0; x < SUB; ++x) r.p[x] = u32x4{0, 0, 0, 0};
                        return r;
                    }
                }
                // Weights are taken against the row's reference, an earlier maximum, as long as no score passes it by more
                // than SLACK: the sums are fp32 and a weight's rounding is relative, so nothing is lost, and the common
                // stage has neither an exchange between lanes nor a rescale.
                float mx = max3(max3(st[0][t][0][0], st[0][t][0][1], st[0][t][0][2]), max3(st[0][t][0][3], st[0][t][1][0], st[0][t][1][1]),
                                max3(st[0][t][1][2], st[0][t][1][3], st[0][t][1][3]));
                if constexpr (SUB == 2)
                    mx = max3(max3(st[1][t][0][0], st[1][t][0][1], st[1][t][0][2]), max3(st[1][t][0][3], st[1][t][1][0], st[1][t][1][1]),
                              max3(st[1][t][1][2], st[1][t][1][3], mx));
                float ref = m_ref[t];
                if (__builtin_amdgcn_ballot_w64(mx > m_lim[t]) != 0) {  // (uniform)
                    const float top = max_x32(max_x16(mx));
                    if (top > m_lim[t] && (top > ref || m_lim[t] == -INFINITY)) {  // (a row's four lanes alike)
                        const float alpha = m_lim[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ref - top) * a.zs);
                        m_ref[t] = ref = top;
                        m_lim[t] = __builtin_fabsf(top * a.zs) > FAR_REF ? -FLT_MAX : top + slack;
                        l[t] *= alpha;
                        if constexpr (WIN) lx[t] *= alpha;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) acc[t][dt] *= alpha;
                    }
                    if (__builtin_amdgcn_ballot_w64(m_lim[t] == -FLT_MAX) != 0) {  // (uniform)
                        const float less = m_lim[t] == -FLT_MAX ? ref : 0.f;
                        ref -= less;
#pragma unroll
                        for (int x = 0; x < SUB; ++x)
#pragma unroll
                            for (int h = 0; h < 2; ++h) st[x][t][h] -= less;
                    }
                }
                const float sub = fmaf(ref, a.zs, -E::SHIFT);
#pragma unroll
                for (int x = 0; x < SUB; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const float p0 = __builtin_amdgcn_exp2f(fmaf(st[x][t][h][i], a.zs, -sub));
                            const float p1 = __builtin_amdgcn_exp2f(fmaf(st[x][t][h][i + 1], a.zs, -sub));
                            r.p[x][2 * h + i / 2] = E::pair(p0, p1);
                            l[t] = E::add_pair(r.p[x][2 * h + i / 2], l[t]);  // (this lane's tokens; the row's four lanes meet at the end)
                            if constexpr (WIN) lx[t] += p0 + p1;
                        }
                return r;
            };
            constexpr int VT = D == 64 ? 4 : 8;  // dim tiles read at once
            u32x2 va[VT], vb[VT];
            // A weight of 0 times an infinity or a NaN in a place that a row does not admit would reach the row: in a stage that
            // not every row admits whole, such values count as 0 here (piece y of the stage). Those that some row of the wave
            // admits it gets when the unit's parts meet, from the stages noted in `odd`. What no row admits (rows behind the
            // last token of a page, the stand-in for a missing page) notes nothing: a cache holds anything there, and the
            // search through a whole share takes milliseconds (a prompt's 2048 rows over 1000, NaN in the unused rows: 103 us as
            // with zeros there, 16.8 ms with every such stage noted and searched from the share's first).
            auto sift = [&](int y) {
                if (!whole) {
                    uint32_t top = 0;
#pragma unroll
                    for (int x = 0; x < VT; ++x)
                        top |= ((va[x].x & E::EXP) + E::ONE) | ((va[x].y & E::EXP) + E::ONE) | ((vb[x].x & E::EXP) + E::ONE) |
                               ((vb[x].y & E::EXP) + E::ONE);
                    if (__builtin_amdgcn_ballot_w64((top & 0x80008000u) != 0) != 0) {
                        // by token: va.x, va.y, vb.x, vb.y hold tokens 4 g, 4 g + 2, 16 + 4 g, 16 + 4 g + 2 and the ones behind
                        auto high = [](uint32_t v) { return ((v & E::EXP) + E::ONE) & 0x80008000u; };
                        auto finite = [&](uint32_t v) { return v & ~((high(v) >> 15) * 0xFFFFu); };
                        uint32_t t0 = 0, t2 = 0, t16 = 0, t18 = 0;
#pragma unroll
                        for (int x = 0; x < VT; ++x) {
                            t0 |= high(va[x].x), t2 |= high(va[x].y), t16 |= high(vb[x].x), t18 |= high(vb[x].y);
                            va[x] = u32x2{finite(va[x].x), finite(va[x].y)};
                            vb[x] = u32x2{finite(vb[x].x), finite(vb[x].y)};
                        }
                        // the piece's tokens that a row of the wave admits (without masks: up to the last row's own)
                        const int p = (WIN ? tree0 : sp.tree0) - v0 - STEP * y;
                        const uint32_t near = WIN ? in_window(r0 + STEP * y, lo_first) : ~0u;
                        uint32_t in;
                        if (a.mask) {
                            uint64_t all = 0;
#pragma unroll
                            for (int t = 0; t < TPW; ++t) all |= bits[t];
#pragma unroll
                            for (int d = 1; d < 16; d <<= 1) all |= __shfl_xor(all, d, 64);
                            const uint64_t own_bits = p >= 32 ? 0 : (p >= 0 ? all << p : (-p < 64 ? all >> -p : 0));
                            in = ((p >= 32 ? ~0u : (p > 0 ? (1u << p) - 1u : 0u)) & near) | uint32_t(own_bits);
                        } else {
                            const int nv = (WIN ? t_none - sp.tree0 + tree0 : t_none) - v0 - STEP * y;
                            in = (nv >= 32 ? ~0u : (nv > 0 ? (1u << nv) - 1u : 0u)) & near;
                        }
                        const uint32_t here = ok >> (2 * y);
                        in &= ((here & 1u) ? 0x0000FFFFu : 0u) | ((here & 2u) ? 0xFFFF0000u : 0u);
                        auto two = [](uint32_t v) { return ((v >> 15) & 1u) | ((v >> 30) & 2u); };
                        const uint32_t found = (two(t0) | (two(t2) << 2) | (two(t16) << 16) | (two(t18) << 18)) << (4 * g);
                        if (__builtin_amdgcn_ballot_w64((found & in) != 0) != 0 && lane == 0) {
                            atomicMin(&odd[0], s);
                            atomicMax(&odd[1], s);
                        }
                    }
                }
            };
            auto weigh = [&](int t, int dt0, u32x4 pf) {
#pragma unroll
                for (int x = 0; x < VT; ++x)
                    acc[t][dt0 + x] = E::mfma(u32x4{va[x].x, va[x].y, vb[x].x, vb[x].y}, pf, acc[t][dt0 + x]);
            };
            auto wait_v = [&]() {
                if constexpr (RTW == 1) {
                    if (more) wait_vm<PER * (2 * NS - 1)>();
                    else wait_vm<0>();
                }
            };
            auto refill_v = [&]() {
                if (RTW == 1 && more) {
                    issue_v(s + AHEAD);
                    next_e = entries(s + AHEAD + 1);
                }
            };
            if constexpr (D != 256 && TPW <= 2 && SUB == 1) {
                // V's reads behind the scores' MFMAs, a tile's products behind the next tile's weights
                wait_v();
                read_v<D, 0>(va, vb, slot + STAGE + v_lane);
                refill_v();
                sift(0);
#pragma unroll
                for (int t = 0; t < TPW; ++t) weigh(t, 0, weights(t).p[0]);
            } else {
                // (V's operands only once the scores' registers are free; at head_dim 256 in halves)
                Weights pf[TPW];
#pragma unroll
                for (int t = 0; t < TPW; ++t) pf[t] = weights(t);
                wait_v();
#pragma unroll
                for (int x = 0; x < SUB; ++x) {
                    read_v<D, 0>(va, vb, slot + STAGE + v_lane + x * STEP * RB);
                    if constexpr (D == 256) {
                        sift(x);
#pragma unroll
                        for (int t = 0; t < TPW; ++t) weigh(t, 0, pf[t].p[x]);
                        read_v<D, 1>(va, vb, slot + STAGE + v_lane);
                    }
                    if (x == SUB - 1) refill_v();
                    sift(x);
#pragma unroll
                    for (int t = 0; t < TPW; ++t) weigh(t, D == 256 ? 8 : 0, pf[t].p[x]);
                }
            }
        }

        // ---- the parts of a row tile meet in LDS, tile by tile; rows D + 4 floats apart (no two rows of an access in one bank)
        const bool first = step0 == 0, last = step0 + nst == n_unit;
        constexpr int OR = D + 4;
        float* const lds_o = reinterpret_cast<float*>(smem);            // [RTW][P][16][OR]
        float* const lm = lds_o + RTW * P * 16 * OR;                    // [RTW][P][16] maxima (log2 units), then sums
        constexpr int MR = RTW * P * 16;
        float* rec = a.part + (int64_t(share) * 2 + (first ? 1 : 0)) * RPW * (D + extra_of(KIND));
        // row r of the unit's block (row s, head h), dims d .. d + 3: done, or to its partial
        auto put = [&](int r, int s, int h, int d, float M, float sum, float sumx, f32x4 o) {
            if (first && last) {
                if (WIN && d == 0) a.lse[(int64_t(b) * a.S + s) * a.H + h] = log_sum<E>(M, sumx);
                const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
                // (no token admitted: 0, whatever o holds)
                *reinterpret_cast<uint2*>(a.out + ((int64_t(b) * a.S + s) * a.H + h) * D + d) =
                    sum == 0.f ? make_uint2(0u, 0u) : make_uint2(E::pair(o[0] * inv, o[1] * inv), E::pair(o[2] * inv, o[3] * inv));
            } else {
                *reinterpret_cast<f32x4*>(rec + int64_t(r) * D + d) = o;
                if (d == 0) {
                    rec[int64_t(RPW) * D + r] = M;
                    rec[int64_t(RPW) * (D + 1) + r] = sum;
                    if (WIN) rec[int64_t(RPW) * (D + 2) + r] = sumx;
                }
            }
        };
        __syncthreads();  // the ring is free
        // The stages are read here alone. A wave that is ahead notes the next unit's without waiting for the others where it has
        // a ring of its own, but not before the barriers below (several parts) or that unit's first stage (waves that share a
        // ring), which a wave that has yet to read them here holds up; so all have one value, as the barriers under it need.
        static_assert(P > 1 || RTW > 1, "");
        const int odd_from = odd[0], odd_to = odd[1];
        const bool left_out = odd_to >= 0;
        // One part: nothing to meet, each lane has its row's four dims of every dim tile (4 x 1024 rows over 1000: 125 us through
        // LDS, 119).
        if (P == 1 && !left_out) {
#pragma unroll
            for (int t = 0; t < TPW; ++t) {
                const int r = (rw * TPW + t) * 16 + c16;
                const float sx = WIN ? sum_x32(sum_x16(lx[t])) : 0.f;
                const float sl = sum_x32(sum_x16(l[t])), M = m_lim[t] == -INFINITY ? -INFINITY : m_ref[t] * a.zs;
                if (r >= rows) continue;
                const int s = s_first + r / a.G, h = kh * a.G + r % a.G;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) put(r, s, h, 16 * dt + 4 * g, M, sl, sx, acc[t][dt]);
            }
        } else {
#pragma unroll
            for (int t = 0; t < TPW; ++t) {
                float* mo = lds_o + (rw * P + part) * 16 * OR + c16 * OR + 4 * g;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(mo + 16 * dt) = acc[t][dt];
                const float sl = sum_x32(sum_x16(l[t])), sx = WIN ? sum_x32(sum_x16(lx[t])) : 0.f;
                if (g == 0) {
                    lm[(rw * P + part) * 16 + c16] = m_lim[t] == -INFINITY ? -INFINITY : m_ref[t] * a.zs;
                    lm[RTW * P * 16 + (rw * P + part) * 16 + c16] = sl;
                    if (WIN) lm[2 * MR + (rw * P + part) * 16 + c16] = sx;
                }
                __syncthreads();
                // thread: row x / (D / 4) of the RTW tiles' 16 each, four dims
                for (int x = tid; x < RTW * 16 * (D / 4); x += NT) {
                    const int rt = x / (16 * (D / 4)), rr = x / (D / 4) % 16, d = x % (D / 4) * 4;
                    const int r = (rt * TPW + t) * 16 + rr;  // row of the unit's block
                    if (r >= rows) continue;
                    const int s = s_first + r / a.G, h = kh * a.G + r % a.G;
                    float M = -INFINITY;
#pragma unroll
                    for (int p = 0; p < P; ++p) M = fmaxf(M, lm[(rt * P + p) * 16 + rr]);
                    float sum = 0.f, sumx = 0.f;
                    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const float mp = lm[(rt * P + p) * 16 + rr];
                        const float wp = mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - M);
                        sum += lm[RTW * P * 16 + (rt * P + p) * 16 + rr] * wp;
                        if (WIN) sumx += lm[2 * MR + (rt * P + p) * 16 + rr] * wp;
                        o += *reinterpret_cast<const f32x4*>(lds_o + (rt * P + p) * 16 * OR + rr * OR + d) * wp;
                    }
                    if (left_out) {  // (what the stages left out, for the rows that admit it)
                        uint64_t own = a.mask ? uint64_t(a.mask[int64_t(b) * a.S + s]) : 0;
                        int lo_row = 0;
                        if constexpr (WIN) {
                            if (a.S < 64) own &= (uint64_t(1) << a.S) - 1;
                            lo_row = sp.n - a.window + (a.mask ? __popcll(own) : s + 1);
                            own = own_in_window(a, own, sp.n);
                        }
                        for (int v = (step0 + odd_from) * TOK; v < min(t_end, (step0 + odd_to + 1) * TOK); ++v) {
                            const int tok = (SEL || WIN) && v >= sp.nsel ? v - sp.nsel + sp.tail : v;
                            const int own_row = WIN ? tok - sp.n : v - sp.tree0;
                            if (own_row >= 0 && !(a.mask ? own_row < 64 && ((own >> own_row) & 1) : own_row <= s)) continue;
                            if (WIN && !(a.mask && own_row >= 0) && tok >= a.first && tok < lo_row) continue;
                            const bool chosen = SEL && v < sp.nsel;
                            if (!chosen && (tok >> a.lt) >= a.W) continue;
                            const int64_t e = chosen ? picked[v >> a.lt] : row[tok >> a.lt];
                            if (e < 0 || e >= a.P) continue;
                            const uint16_t* src = a.value + kh * a.vh + e * a.vp + (tok & ((1 << a.lt) - 1)) * a.vt + d;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float x = E::to_f32(src[i]);
                                if (!(__builtin_fabsf(x) < INFINITY)) o[i] += x;
                            }
                        }
                    }
                    put(r, s, h, d, M, sum, sumx, o);
                }
                __syncthreads();
            }
        }
        if (first && tid == 0 && !a.whole && (a.by_unit || !last)) {
            // the unit goes on in the shares behind: how many in all (1: it is done)
            const int unit = (b * a.Hk + kh) * a.units + u, left = n_unit - nst;
            a.info[a.by_unit ? unit : share] = make_int4(unit, share, 1 + (left + quota - 1) / quota, 0);
        }

        // ---- the next unit
        at += nst + (last ? Geo::FIXED : 0);
        if (at >= end) break;
        if (left_out) {  // (uniform)
            if (tid == 0) odd[0] = INT_MAX, odd[1] = -1;  // (every wave has read it: the barriers of the meeting lie between)
            __syncthreads();
        }
        step0 = 0;
        next_unit();
    }
}

// The units that several shares worked on: a wave per query row (four rows one after the other where there are many:
// 37 us against 20 for 64 blocks of 128). D / 4 lanes take a partial's row in 16-byte pieces, 256 / D partials at
// once; the maxima, sums and pieces of up to eight each go out together, so that few partials cost one memory round trip
// behind the share's entry.
template <class E, int D, Kind KIND>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int rpw) {
    constexpr bool WIN = KIND == Kind::WIN;
    const int4 x = a.info[blockIdx.x];
    const int nseg = x.z, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (nseg <= 1) return;
    const int u = x.x % a.units, kh = x.x / a.units % a.Hk, b = x.x / a.units / a.Hk;
    constexpr int TPR = D / 4, NG = 64 / TPR, U = 8;
    const int gi = lane / TPR, d = lane % TPR * 4;
    const int64_t rec = int64_t(rpw) * (D + extra_of(KIND));
    const float* base = a.part + int64_t(x.y) * 2 * rec;
    const int r = int(blockIdx.y) * 4 + w, s = u * a.spb + r / a.G, h = kh * a.G + r % a.G;
    if (r >= a.spb * a.G || s >= a.S) return;  // (uniform in the wave)
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, sum = 0.f, sumx = 0.f;
    for (int i0 = 0; i0 < nseg; i0 += U * NG) {
        f32x4 v[U];
        float mi[U], li[U], xi[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int sg = min(i0 + i * NG + gi, nseg - 1);  // (past the last: read again, not counted)
            const float* p = base + (sg == 0 ? 1 : 2 * sg) * rec;
            mi[i] = p[int64_t(rpw) * D + r];
            li[i] = p[int64_t(rpw) * (D + 1) + r];
            if (WIN) xi[i] = p[int64_t(rpw) * (D + 2) + r];
            v[i] = *reinterpret_cast<const f32x4*>(p + int64_t(r) * D + d);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (i0 + i * NG + gi >= nseg) mi[i] = -INFINITY;
            top = fmaxf(top, mi[i]);
        }
        const float was = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
        o *= was;
        sum *= was;
        if (WIN) sumx *= was;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (i0 + i * NG + gi >= nseg) continue;
            // (a partial without an admitted token has sum 0 and O 0)
            const float wi = mi[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi[i] - top);
            sum += li[i] * wi;
            if (WIN) sumx += xi[i] * wi;
            o += v[i] * wi;
        }
        M = top;
    }
    float top = M;
#pragma unroll
    for (int j = TPR; j < 64; j <<= 1) top = fmaxf(top, __shfl_xor(top, j, 64));
    const float own = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
    o *= own;
    sum *= own;
    if (WIN) sumx *= own;
#pragma unroll
    for (int j = TPR; j < 64; j <<= 1) {
        sum += __shfl_xor(sum, j, 64);
        if (WIN) sumx += __shfl_xor(sumx, j, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], j, 64);
    }
    if (gi != 0) return;
    if (WIN && d == 0) a.lse[(int64_t(b) * a.S + s) * a.H + h] = log_sum<E>(top, sumx);
    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
    *reinterpret_cast<uint2*>(a.out + ((int64_t(b) * a.S + s) * a.H + h) * D + d) =
        sum == 0.f ? make_uint2(0u, 0u) : make_uint2(E::pair(o[0] * inv, o[1] * inv), E::pair(o[2] * inv, o[3] * inv));
}

// ---- the selection ----------------------------------------------------------------------------------------
// Scores of the full pages between the forced ones: (sum of the group's queries) . mean key, in float64 (the order of
// scores decides, and 32-bit sums in another order would swap neighbours), as keys whose unsigned order is the scores'
// (NaN lowest). Products of 16 rows and 16 pages by v_mfma_f64_16x16x4 (A: lane (row c16, k g), B: lane (page c16, k g),
// the four dims of a product being dim e of the four 8-dim pieces that the lanes of a page hold; D: lane (row 4 r + g, page
// c16) in element r): a wave takes 16 pages, so the longest context spreads over all CUs. (One thread per page on the vector
// units: 94.8 us for 8 rows over 250 pages of head_dim 256, 21 us for 1 row over 2046 of 128.)
constexpr int SCORE_ROWS = 16;
// Rows up to which the vector units take them, an MFMA of one row taking as long as of 16 (a call with one row over 60000
// pages: 115 us, 124 by MFMA; 16 x 1 over 500: 43.6 and 46.9; 4 rows over 2046: 31.0 and 30.4; 8: 37.4 and 34.9).
constexpr int FEW_ROWS = 2;
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
template <class E, int D>
__global__ __launch_bounds__(256) void block_score_kernel(PagedArgs a) {
    constexpr int QR = D + 2;  // (rows two doubles further apart: no bank conflicts)
    __shared__ __align__(16) double qs[SCORE_ROWS * QR];
    const int b = blockIdx.z / a.Hk, kh = blockIdx.z % a.Hk, s0 = blockIdx.y * SCORE_ROWS, ns = min(SCORE_ROWS, a.S - s0);
    const int c = span_of<Kind::SEL>(a, a.length[b], 0).tail >> a.lt, j_end = c - a.local;
    if (c <= a.most || a.sink + int(blockIdx.x) * 64 >= j_end) return;  // (uniform: all pages are selected, or none is scored here)
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const int j = a.sink + int(blockIdx.x) * 64 + int(threadIdx.x >> 6) * 16 + c16;
    const int e = j < j_end ? a.table[b * a.ts + j] : -1;
    const bool in = e >= 0 && e < a.P;
    u32x4 k[D / 32];  // (the page's mean key goes out ahead of the queries; a page that is none reads page 0)
    const uint16_t* kp = a.ksum + kh * a.sh + (in ? e : 0) * a.sp + 8 * g;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) k[i] = *reinterpret_cast<const u32x4*>(kp + 32 * i);
    for (int i = threadIdx.x; i < ns * (D / 8); i += 256) {  // (eight dims each: one round of loads for 8 rows of 256)
        const int s = i / (D / 8), d = i % (D / 8) * 8;
        const uint16_t* p = a.q + b * a.qb + (s0 + s) * a.qs + kh * a.G * a.qh + d;
        double t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
        for (int h = 0; h < a.G; ++h) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p + h * a.qh);
#pragma unroll
            for (int x = 0; x < 8; ++x) t[x] += double(E::to_f32(uint16_t(v[x / 2] >> (16 * (x & 1)))));
        }
#pragma unroll
        for (int x = 0; x < 8; x += 2) *reinterpret_cast<f64x2*>(qs + s * QR + d + x) = f64x2{t[x], t[x + 1]};
    }
    __syncthreads();
    auto put = [&](int s, double z) {
        z += 0.0;  // (-0 and 0 are one score)
        const uint64_t x = __builtin_bit_cast(uint64_t, z);
        a.keys[((int64_t(b) * a.S + s0 + s) * a.Hk + kh) * a.W + j] = !in || z != z ? 0 : (x >> 63 ? ~x : x | (uint64_t(1) << 63));
    };
    if (ns <= FEW_ROWS) {  // (uniform)
        double kd[D / 4];
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int x = 0; x < 8; ++x) kd[8 * i + x] = double(E::to_f32(uint16_t(k[i][x / 2] >> (16 * (x & 1)))));
        for (int s = 0; s < ns; ++s) {
            const double* q = qs + s * QR + 8 * g;
            double t0 = 0, t1 = 0;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f64x2 qq = *reinterpret_cast<const f64x2*>(q + 32 * i + 2 * x);
                    t0 = fma(qq[0], kd[8 * i + 2 * x], t0);
                    t1 = fma(qq[1], kd[8 * i + 2 * x + 1], t1);
                }
            t0 += t1;
            t0 += __shfl_xor(t0, 16, 64);
            t0 += __shfl_xor(t0, 32, 64);
            if (g == 0 && j < j_end) put(s, t0);
        }
        return;
    }
    const double* q = qs + min(c16, ns - 1) * QR + 8 * g;  // (rows past the last repeat it: their products are not written)
    f64x4 dot = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const f64x2 qq = *reinterpret_cast<const f64x2*>(q + 32 * i + 2 * x);
            dot = __builtin_amdgcn_mfma_f64_16x16x4f64(qq[0], double(E::to_f32(uint16_t(k[i][x] & 0xFFFFu))), dot, 0, 0, 0);
            dot = __builtin_amdgcn_mfma_f64_16x16x4f64(qq[1], double(E::to_f32(uint16_t(k[i][x] >> 16))), dot, 0, 0, 0);
        }
    if (j >= j_end) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4 * r + g < ns) put(4 * r + g, dot[r]);
}

__device__ __forceinline__ int wave_incl_sum(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d, 64);
        if (lane >= d) v += u;
    }
    return v;
}

// The `blocks` best of the scored pages (ties to the lowest index) and the forced ones, ascending: one work-group per
// (sequence, row, kv head), the keys in registers (W <= NT EACH; past 16 per thread they are read again). The threshold: a
// histogram of 1024 bins, even steps between the lowest and the highest score (in fp32: rounding keeps their order), then
// the keys of the one bin that holds it by their ranks; where that bin has more than NT keys (ties, or an infinity that
// stretches the range), by bytes from the top instead. Then one pass in index order. Bound by latency (barriers and LDS): 9 us
// with a byte-wise threshold and a barrier pair per NT keys of the last pass, at 2046 pages.
template <int NT, int EACH>
__global__ __launch_bounds__(NT) void block_select_kernel(PagedArgs a) {
    constexpr int NW = NT / 64, BINS = 1024;
    constexpr bool REG = EACH <= 16;
    constexpr int U = REG ? EACH : 1;
    __shared__ int hist[BINS];
    __shared__ int tmp[NW], pick[3], found;
    __shared__ float lo_w[NW], hi_w[NW];
    __shared__ uint64_t cand[NT], thr;
    __shared__ int pre[2][NW * EACH];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t unit = blockIdx.x;
    const int b = int(unit / (int64_t(a.S) * a.Hk));
    const int c = span_of<Kind::SEL>(a, a.length[b], 0).tail >> a.lt;
    int32_t* sel = a.sel + unit * a.most;
    int32_t* page = a.page + unit * a.most;
    const int32_t* row = a.table + b * a.ts;
    if (c <= a.most) {  // every full page
        for (int i = tid; i < a.most; i += NT) {
            sel[i] = i < c ? i : -1;
            page[i] = i < c ? row[i] : -1;
        }
        return;
    }
    const int j0 = a.sink, j1 = c - a.local, want = a.most - a.sink - a.local;
    for (int i = tid; i < a.sink; i += NT) {
        sel[i] = i;
        page[i] = row[i];
    }
    for (int i = tid; i < a.local; i += NT) {
        sel[a.sink + want + i] = j1 + i;
        page[a.sink + want + i] = row[j1 + i];
    }
    if (want == 0) return;
    const uint64_t* keys = a.keys + unit * a.W;
    uint64_t kept[U];
    float lo = INFINITY, hi = -INFINITY;
    if constexpr (REG)
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int j = j0 + i * NT + tid;
            kept[i] = j < j1 ? keys[j] : 0;
        }
    auto live = [&](int i) { return j0 + i * NT + tid < j1; };
    auto key = [&](int i) -> uint64_t {
        if constexpr (REG) return kept[i];
        return live(i) ? keys[j0 + i * NT + tid] : 0;
    };
    // a key's score in fp32, a quarter of it (the range stays finite); a NaN's is the lowest there is
    auto score = [](uint64_t x) {
        if (x == 0) return -0.25f * 3.402823466e38f;
        const double d = __builtin_bit_cast(double, x >> 63 ? x & ~(uint64_t(1) << 63) : ~x);
        return 0.25f * fminf(fmaxf(float(d), -3.402823466e38f), 3.402823466e38f);
    };
#pragma unroll U
    for (int i = 0; i < EACH; ++i)
        if (live(i)) {
            const float x = score(key(i));
            lo = fminf(lo, x);
            hi = fmaxf(hi, x);
        }
    for (int d = 32; d; d >>= 1) {
        lo = fminf(lo, __shfl_xor(lo, d, 64));
        hi = fmaxf(hi, __shfl_xor(hi, d, 64));
    }
    for (int i = tid; i < BINS; i += NT) hist[i] = 0;
    if (lane == 0) {
        lo_w[w] = lo;
        hi_w[w] = hi;
    }
    if (tid == 0) found = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        lo = fminf(lo, lo_w[i]);
        hi = fmaxf(hi, hi_w[i]);
    }
    const float per = hi - lo > 1e-30f ? float(BINS - 1) / (hi - lo) : 0.f;
    auto bin = [&](uint64_t x) { return int(fminf((score(x) - lo) * per, float(BINS - 1))); };
#pragma unroll U
    for (int i = 0; i < EACH; ++i)
        if (live(i)) atomicAdd(&hist[bin(key(i))], 1);
    __syncthreads();
    // the bin that holds the want-th key from the top
    {
        constexpr int PB = BINS / NT;  // bins per thread, from the top
        int sum = 0;
#pragma unroll
        for (int i = 0; i < PB; ++i) sum += hist[BINS - 1 - (tid * PB + i)];
        const int incl = wave_incl_sum(sum, lane);
        if (lane == 63) tmp[w] = incl;
        __syncthreads();
        int before = incl - sum;
        for (int i = 0; i < w; ++i) before += tmp[i];
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            const int x = hist[BINS - 1 - (tid * PB + i)];
            if (before < want && before + x >= want) {
                pick[0] = BINS - 1 - (tid * PB + i);
                pick[1] = want - before;
                pick[2] = x;
            }
            before += x;
        }
    }
    __syncthreads();
    const int at_bin = pick[0], in_bin = pick[2];
    int left = pick[1], shift = 0;
    uint64_t prefix;
    if (in_bin <= NT) {
#pragma unroll U
        for (int i = 0; i < EACH; ++i)
            if (live(i) && bin(key(i)) == at_bin) cand[atomicAdd(&found, 1)] = key(i);
        __syncthreads();
        if (tid < in_bin) {  // (equal keys find the same threshold and count: whichever thread writes last)
            const uint64_t mine = cand[tid];
            int above = 0, same = 0;
            for (int i = 0; i < in_bin; ++i) {
                above += cand[i] > mine;
                same += cand[i] == mine;
            }
            if (above < left && left <= above + same) {
                thr = mine;
                pick[1] = left - above;
            }
        }
        __syncthreads();
        prefix = thr;
        left = pick[1];
    } else {
        // by bytes, among the keys of that bin; `left` of them are wanted
        prefix = 0;
        shift = 64;
        bool exact = false;  // every key of the last byte's value is taken
        while (!exact && shift > 0) {
            shift -= 8;
            __syncthreads();
            for (int i = tid; i < 256; i += NT) hist[i] = 0;
            __syncthreads();
#pragma unroll U
            for (int i = 0; i < EACH; ++i)
                if (live(i) && bin(key(i)) == at_bin && (shift == 56 || (key(i) >> (shift + 8)) == prefix))
                    atomicAdd(&hist[int(key(i) >> shift) & 255], 1);
            __syncthreads();
            if (w == 0) {  // four bytes' values per lane, from 255 downwards
                int v[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += v[i] = hist[255 - (lane * 4 + i)];
                int before = wave_incl_sum(sum, lane) - sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < left && before + v[i] >= left) {
                        pick[0] = 255 - (lane * 4 + i);
                        pick[1] = left - before;
                        pick[2] = v[i];
                    }
                    before += v[i];
                }
            }
            __syncthreads();
            prefix = (prefix << 8) | uint64_t(pick[0]);
            left = pick[1];
            exact = pick[2] == left;
        }
    }
    // keys above the threshold (a higher bin, or its bin and higher in the bytes above `shift`), and `left` of those at it, the
    // first in index order
    auto side = [&](int i) { return !live(i) || bin(key(i)) < at_bin ? 0 : bin(key(i)) > at_bin || (key(i) >> shift) > prefix ? 2 : (key(i) >> shift) == prefix ? 1 : 0; };
#pragma unroll U
    for (int i = 0; i < EACH; ++i) {
        const int x = side(i);
        const uint64_t above = __builtin_amdgcn_ballot_w64(x == 2), ties = __builtin_amdgcn_ballot_w64(x == 1);
        if (lane == 0) {
            pre[0][i * NW + w] = __popcll(above);
            pre[1][i * NW + w] = __popcll(ties);
        }
    }
    __syncthreads();
    if (w < 2) {  // exclusive sums over (i, wave), in index order
        int carry = 0;
        for (int r = 0; r < NW * EACH; r += 64) {
            const int x = r + lane < NW * EACH ? pre[w][r + lane] : 0;
            const int incl = wave_incl_sum(x, lane);
            if (r + lane < NW * EACH) pre[w][r + lane] = carry + incl - x;
            carry += __shfl(incl, 63, 64);
        }
    }
    __syncthreads();
    const uint64_t under = (uint64_t(1) << lane) - 1;
#pragma unroll U
    for (int i = 0; i < EACH; ++i) {
        const int x = side(i);
        const uint64_t above = __builtin_amdgcn_ballot_w64(x == 2), tie = __builtin_amdgcn_ballot_w64(x == 1);
        const int ties = pre[1][i * NW + w] + __popcll(tie & under);
        if (x == 2 || (x == 1 && ties < left)) {
            const int j = j0 + i * NT + tid, to = a.sink + pre[0][i * NW + w] + __popcll(above & under) + min(ties, left);
            sel[to] = j;
            page[to] = row[j];
        }
    }
}

// ---- launches ---------------------------------------------------------------------------------------------
// The most tokens a unit can have: all that the table (or a selection) holds, and the rows' own; in a window, that of its rows
// and the first tokens, in whole stages.
int64_t window_tokens(int64_t held, int64_t S, int64_t spb, int64_t window, int64_t first) {
    const int64_t rows = S < 64 ? S : spb > 64 ? spb : 64, heads = (first + WIN_STEP - 1) / WIN_STEP * WIN_STEP;
    const int64_t most = heads + window + (rows < S ? rows : S) + WIN_STEP - 1;
    return most < held + S ? most : held + S;
}
template <Kind KIND>
int64_t most_tokens(const PagedArgs& a) {
    if (KIND == Kind::WIN) return window_tokens(int64_t(a.W) << a.lt, a.S, a.spb, a.window, a.first);
    const int64_t pages = KIND == Kind::SEL && a.most < a.W ? a.most + 1 : a.W;
    return (pages << a.lt) + a.S;
}

template <class E, int D, int TPW, int RTW, int P, int WPC, Kind KIND, int SUB = 1>
int launch(PagedArgs& a, hipStream_t st) {
    using Geo = Geometry<D, TPW, RTW, P, WPC, SUB>;
    constexpr int joined = (RTW * P * 16 * (D + 4) + extra_of(KIND) * RTW * P * 16) * 4;
    constexpr int lds = Geo::RING > joined ? Geo::RING : joined;
    // (once per device and kernel: the call costs about a microsecond)
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    MDX_HIP(hipGetDevice(&dev));
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (dev > 63 || !(allowed.load(std::memory_order_relaxed) & bit)) {
        allow_smem(reinterpret_cast<const void*>(&paged_attn_kernel<E, D, TPW, RTW, P, WPC, SUB, KIND>), lds);
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    // Row blocks enough for every work-group there is room for: whole ones, without partials, as long as no unit can be much
    // longer than the others (2048 rows over 1000 tokens: 122 us in shares, 90 whole; 16 x 128 rows over 1000 each: 87 and 52;
    // over 0 to 6000: 166 and 161; but with one sequence of 60000 among 15 of 500: 211 and 1437).
    const int units = a.B * a.Hk * a.units;
    const int64_t most = most_tokens<KIND>(a);
    if (a.units > 1 && units >= CUS * WPC && (a.B == 1 || most <= EVEN_TOKENS || int64_t(units) * a.S >= most * CUS * WPC)) a.whole = 1;
    const int grid = a.whole ? units : CUS * WPC;
    a.by_unit = units <= grid;  // (every unit is begun by one share, which writes its entry)
    hipLaunchKernelGGL((paged_attn_kernel<E, D, TPW, RTW, P, WPC, SUB, KIND>), dim3(unsigned(grid)), dim3(Geo::NT), lds, st, a);
    MDX_LAUNCHED();
    if (a.whole) return MDX_OK;
    const int rows = (a.spb < a.S ? a.spb : a.S) * a.G;
    hipLaunchKernelGGL((paged_join_kernel<E, D, KIND>), dim3(unsigned(units < grid ? units : grid), unsigned((rows + 3) / 4)), dim3(256), 0, st, a,
                       Geo::RPW);
    MDX_LAUNCHED();
    return MDX_OK;
}

// Query rows of a work-group: what covers the rows of a kv head with as few row blocks as registers allow.
int rpw_of(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

// The form by the rows of a unit. A unit's row tiles lie in waves of their own, which read each K and V operand from LDS again
// but have fewer instructions one after the other (32 and 64 rows in one wave's registers: 20 against 15 us for 16 rows over
// 1000 tokens of 8 kv heads, 120 against 106 for 16 sequences over 8000); only at head_dim 64 LDS is what bounds 64 rows where
// there is much to stream (32 sequences of 16 rows over 8000: 106 us in one wave's registers, 117 in waves of their own).
template <class E, int D, Kind KIND>
int launch_rows(PagedArgs& a, hipStream_t st) {
    constexpr bool SEL = KIND == Kind::SEL;
    const int rows = SEL ? a.G : a.units > 1 ? 128 : a.S * a.G;
    const int64_t steps = int64_t(a.B) * a.Hk * a.units * ((most_tokens<KIND>(a) + 127) / 128);
    const bool few = steps <= FEW_STEPS;
    // Two work-groups per CU where there is much to stream: one goes on while the other changes units (16 x 8 rows' selections
    // of 16 blocks: 121 -> 109 us, 200 single tokens over 10 to 500: 50 -> 46, 64 over at most 8192 at head_dim 64: 98 -> 93, at
    // 128: 195 -> 198; one token over 2000: 11.7 -> 12.1; at head_dim 256 a stage of 32 KiB leaves no ring for it).
    if (rows <= 16) {
        if (few || D == 256) return launch<E, D, 1, 1, 4, 1, KIND>(a, st);
        if constexpr (D != 256) return launch<E, D, 1, 1, 4, 2, KIND>(a, st);
    }
    if (rows <= 32) return launch<E, D, 1, 2, (D == 256 ? 2 : 4), 1, KIND>(a, st);
    if (rows <= 64) {
        if constexpr (D == 64)
            if (!few) return launch<E, D, 4, 1, 4, 1, KIND>(a, st);
        return launch<E, D, 1, 4, (D == 256 ? 1 : 2), 1, KIND>(a, st);
    }
    if constexpr (!SEL) return launch<E, D, 2, 4, 1, (D == 256 ? 1 : 2), KIND, (D == 256 ? 1 : 2)>(a, st);
    set_error("at most 64 query heads per kv head");
    return MDX_EINVAL;
}

template <Kind KIND>
int launch_any(PagedArgs& a, int D, int dtype, hipStream_t st) {
    if (dtype == MDX_DT_BF16) {
        if (D == 64) return launch_rows<Bf16, 64, KIND>(a, st);
        if (D == 128) return launch_rows<Bf16, 128, KIND>(a, st);
        return launch_rows<Bf16, 256, KIND>(a, st);
    }
    if (D == 64) return launch_rows<Fp16, 64, KIND>(a, st);
    if (D == 128) return launch_rows<Fp16, 128, KIND>(a, st);
    return launch_rows<Fp16, 256, KIND>(a, st);
}

size_t base_bytes(int64_t rows, int64_t D, Kind kind) {
    const int rpw = rpw_of(rows), shares = rpw == 16 || rpw == 128 ? 2 * CUS : CUS;
    return size_t(2 * CUS) * sizeof(int4) + size_t(shares) * 2 * rpw * (D + extra_of(kind)) * 4;
}

int log2_of(int64_t T) {
    for (int i = 4; i <= 10; ++i)
        if (T == int64_t(1) << i) return i;
    return -1;
}

// what both entry points check and set
int fill(PagedArgs& a, const void* q, int64_t q_seq_stride, int64_t q_row_stride, int64_t q_head_stride, const void* key,
         int64_t k_head_stride, int64_t k_page_stride, int64_t k_row_stride, const void* value, int64_t v_head_stride,
         int64_t v_page_stride, int64_t v_row_stride, int32_t dtype, const int32_t* table, int64_t table_stride,
         const int32_t* length, const int64_t* mask, void* out, int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D,
         int64_t P, int64_t T, int64_t W, float scale) {
    MDX_CHECK(q && key && value && table && length && out, "null pointer");
    MDX_CHECK(dtype == MDX_DT_BF16 || dtype == MDX_DT_F16, "bf16 or fp16");
    MDX_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
    const int lt = log2_of(T);
    MDX_CHECK(lt >= 0, "page rows: a power of two in 16..1024");
    MDX_CHECK(B >= 1 && B <= MAX_SEQS && Hk >= 1 && Hk <= 1024 && H >= 1 && H % Hk == 0 && H <= 65536, "1..1024 sequences, heads");
    MDX_CHECK(P >= 1 && P <= (int64_t(1) << 30) && W >= 1 && (W << lt) < (int64_t(1) << 30) && table_stride >= W &&
                  table_stride <= (int64_t(1) << 26),
              "pages, table [sequences, W], under 2^30 tokens a sequence");
    const int64_t lim = int64_t(1) << 40;
    MDX_CHECK(k_row_stride >= D && v_row_stride >= D && k_row_stride <= (int64_t(1) << 24) && v_row_stride <= (int64_t(1) << 24) &&
                  k_head_stride >= 0 && v_head_stride >= 0 && k_page_stride >= 0 && v_page_stride >= 0 && k_head_stride < lim &&
                  v_head_stride < lim && k_page_stride < lim && v_page_stride < lim,
              "cache strides (rows of D elements or further apart)");
    MDX_CHECK(aligned(q, 16) && aligned(key, 16) && aligned(value, 16) && aligned(out, 8) && q_seq_stride % 8 == 0 &&
                  q_row_stride % 8 == 0 && q_head_stride % 8 == 0 && k_head_stride % 8 == 0 && k_page_stride % 8 == 0 &&
                  k_row_stride % 8 == 0 && v_head_stride % 8 == 0 && v_page_stride % 8 == 0 && v_row_stride % 8 == 0,
              "16-byte aligned rows");
    MDX_CHECK(scale > 0.f && scale < INFINITY, "a positive, finite scale");
    MDX_CHECK(q_seq_stride >= 0 && q_row_stride >= 0 && q_head_stride >= 0 && q_seq_stride < lim && q_row_stride < lim && q_head_stride < lim,
              "query strides");
    // (a row is written while work-groups that have a part of it may still have its query to read)
    const uint64_t q_bytes = uint64_t((B - 1) * q_seq_stride + (S - 1) * q_row_stride + (H - 1) * q_head_stride + D) * 2;
    MDX_CHECK(apart(out, uint64_t(B * S * H * D) * 2, q, q_bytes), "out: apart from q");
    a.q = static_cast<const uint16_t*>(q);
    a.qb = q_seq_stride, a.qs = q_row_stride, a.qh = q_head_stride;
    a.key = static_cast<const uint16_t*>(key);
    a.kh = k_head_stride, a.kp = k_page_stride, a.kt = k_row_stride;
    a.value = static_cast<const uint16_t*>(value);
    a.vh = v_head_stride, a.vp = v_page_stride, a.vt = v_row_stride;
    a.table = table;
    a.ts = table_stride;
    a.length = length;
    a.mask = mask;
    a.out = static_cast<uint16_t*>(out);
    a.B = int(B), a.S = int(S), a.H = int(H), a.Hk = int(Hk), a.G = int(H / Hk), a.W = int(W), a.P = int(P), a.lt = lt;
    a.zs = float(double(scale) * 1.4426950408889634);
    return MDX_OK;
}

}  // namespace
}  // namespace mdx

using namespace mdx;

// Rows s of a unit (a work-group's rows hold whole groups of heads), and a kv head's units.
static int64_t rows_of_unit(int64_t S, int64_t G) { return rpw_of(S * G) / G; }
static int64_t blocks_of(int64_t S, int64_t G) { return G > 128 ? 0 : (S + rows_of_unit(S, G) - 1) / rows_of_unit(S, G); }

// One work-group per unit, without a join: where a unit has few steps at most.
static bool whole_units(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t most) {
    const int64_t units = B * Hk * blocks_of(S, H / Hk);
    return most <= (2 * units >= CUS && units <= CUS ? 2 : 1) * WHOLE_TOKENS && units <= 65536;
}

extern "C" size_t mdx_attn_paged_workspace(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t T, int64_t W) {
    if (B < 1 || S < 1 || Hk < 1 || H < 1 || H % Hk != 0 || D < 1 || T < 1 || W < 1 || W > (int64_t(1) << 30)) return 0;
    return whole_units(B, S, H, Hk, W * T + S) ? 0 : base_bytes(S * (H / Hk), D, Kind::ALL);
}

extern "C" int mdx_attn_paged(const void* q, int64_t q_seq_stride, int64_t q_row_stride, int64_t q_head_stride, const void* key,
                              int64_t k_head_stride, int64_t k_page_stride, int64_t k_row_stride, const void* value,
                              int64_t v_head_stride, int64_t v_page_stride, int64_t v_row_stride, int32_t dtype,
                              const int32_t* table, int64_t table_stride, const int32_t* length, const int64_t* mask, void* out,
                              int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t P, int64_t T, int64_t W,
                              float scale, void* workspace, size_t workspace_bytes, void* stream) {
    MDX_CHECK(S >= 1 && (mask ? S <= 64 : S <= 65535), "1..64 rows with masks, 1..65535 without");
    PagedArgs a{};
    const int rc = fill(a, q, q_seq_stride, q_row_stride, q_head_stride, key, k_head_stride, k_page_stride, k_row_stride, value,
                        v_head_stride, v_page_stride, v_row_stride, dtype, table, table_stride, length, mask, out, B, S, H, Hk, D, P,
                        T, W, scale);
    if (rc != MDX_OK) return rc;
    MDX_CHECK(H / Hk <= 128, "at most 128 query heads per kv head");
    const int64_t rows = S * (H / Hk), blocks = blocks_of(S, H / Hk);
    MDX_CHECK(rows < (int64_t(1) << 30) && B * Hk * blocks < (int64_t(1) << 30) && B * Hk * blocks * ((W * T + S) / STEP + 8) < MAX_LINE,
              "too many rows times tokens for one call");
    a.whole = whole_units(B, S, H, Hk, W * T + S);
    MDX_CHECK(a.whole || (workspace && aligned(workspace, 16) && workspace_bytes >= base_bytes(rows, D, Kind::ALL)),
              "workspace: %zu bytes, 16-byte aligned", base_bytes(rows, D, Kind::ALL));
    a.spb = int(rows_of_unit(S, H / Hk));
    a.units = int(blocks);
    a.info = static_cast<int4*>(workspace);
    a.part = reinterpret_cast<float*>(a.info + 2 * CUS);
    return launch_any<Kind::ALL>(a, int(D), dtype, static_cast<hipStream_t>(stream));
}

extern "C" size_t mdx_attn_window_workspace(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t T, int64_t W,
                                            int64_t window, int64_t sinks) {
    if (B < 1 || S < 1 || Hk < 1 || H < 1 || H % Hk != 0 || H / Hk > 128 || D < 1 || T < 1 || W < 1 || W > (int64_t(1) << 30) || window < 1 ||
        sinks < 0 || window > (int64_t(1) << 30) || sinks > (int64_t(1) << 30))
        return 0;
    const int64_t most = window_tokens(W * T, S, rows_of_unit(S, H / Hk), window, sinks);
    return whole_units(B, S, H, Hk, most) ? 0 : base_bytes(S * (H / Hk), D, Kind::WIN);
}

extern "C" int mdx_attn_window(const void* q, int64_t q_seq_stride, int64_t q_row_stride, int64_t q_head_stride, const void* key,
                               int64_t k_head_stride, int64_t k_page_stride, int64_t k_row_stride, const void* value,
                               int64_t v_head_stride, int64_t v_page_stride, int64_t v_row_stride, int32_t dtype,
                               const int32_t* table, int64_t table_stride, const int32_t* length, const int64_t* mask, void* out,
                               float* lse, int64_t window, int64_t sinks, int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D,
                               int64_t P, int64_t T, int64_t W, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    MDX_CHECK(S >= 1 && (mask ? S <= 64 : S <= 65535), "1..64 rows with masks, 1..65535 without");
    MDX_CHECK(lse && aligned(lse, 4), "null pointer");
    MDX_CHECK(window >= 1 && window <= (int64_t(1) << 30) && sinks >= 0 && sinks <= (int64_t(1) << 30), "a window of 1..2^30 tokens, 0..2^30 first ones");
    PagedArgs a{};
    const int rc = fill(a, q, q_seq_stride, q_row_stride, q_head_stride, key, k_head_stride, k_page_stride, k_row_stride, value,
                        v_head_stride, v_page_stride, v_row_stride, dtype, table, table_stride, length, mask, out, B, S, H, Hk, D, P,
                        T, W, scale);
    if (rc != MDX_OK) return rc;
    MDX_CHECK(H / Hk <= 128, "at most 128 query heads per kv head");
    const int64_t rows = S * (H / Hk), blocks = blocks_of(S, H / Hk), most = window_tokens(W * T, S, rows_of_unit(S, H / Hk), window, sinks);
    MDX_CHECK(rows < (int64_t(1) << 30) && B * Hk * blocks < (int64_t(1) << 30) && B * Hk * blocks * (most / STEP + 8) < MAX_LINE,
              "too many rows times tokens for one call");
    a.whole = whole_units(B, S, H, Hk, most);
    MDX_CHECK(a.whole || (workspace && aligned(workspace, 16) && workspace_bytes >= base_bytes(rows, D, Kind::WIN)),
              "workspace: %zu bytes, 16-byte aligned", base_bytes(rows, D, Kind::WIN));
    // (written while other rows' outputs and queries are)
    const uint64_t q_bytes = uint64_t((B - 1) * q_seq_stride + (S - 1) * q_row_stride + (H - 1) * q_head_stride + D) * 2, l_bytes = uint64_t(B * S * H) * 4;
    MDX_CHECK(apart(lse, l_bytes, out, uint64_t(B * S * H * D) * 2) && apart(lse, l_bytes, q, q_bytes), "lse: apart from out and q");
    a.spb = int(rows_of_unit(S, H / Hk));
    a.units = int(blocks);
    a.first = int(sinks), a.window = int(window);
    a.lse = lse;
    a.info = static_cast<int4*>(workspace);
    a.part = reinterpret_cast<float*>(a.info + 2 * CUS);
    return launch_any<Kind::WIN>(a, int(D), dtype, static_cast<hipStream_t>(stream));
}

extern "C" size_t mdx_attn_blocks_workspace(int64_t B, int64_t S, int64_t H, int64_t Hk, int64_t D, int64_t W, int64_t most) {
    if (B < 1 || S < 1 || Hk < 1 || H < 1 || H % Hk != 0 || D < 1 || W < 1 || most < 1) return 0;
    return base_bytes(H / Hk, D, Kind::SEL) + size_t(B * S * Hk) * (size_t(W) * 8 + size_t((most + 3) / 4 * 4) * 4);
}

extern "C" int mdx_attn_blocks(const void* q, int64_t q_seq_stride, int64_t q_row_stride, int64_t q_head_stride, const void* key,
                               int64_t k_head_stride, int64_t k_page_stride, int64_t k_row_stride, const void* value,
                               int64_t v_head_stride, int64_t v_page_stride, int64_t v_row_stride, const void* ksum,
                               int64_t s_head_stride, int64_t s_page_stride, int32_t dtype, const int32_t* table,
                               int64_t table_stride, const int32_t* length, const int64_t* mask, void* out, int32_t* sel,
                               int64_t blocks, int64_t sink, int64_t local, int64_t B, int64_t S, int64_t H, int64_t Hk,
                               int64_t D, int64_t P, int64_t T, int64_t W, float scale, void* workspace, size_t workspace_bytes,
                               void* stream) {
    MDX_CHECK(S >= 1 && S <= 64, "1..64 rows");
    MDX_CHECK(ksum && sel, "null pointer");
    MDX_CHECK(blocks >= 0 && sink >= 0 && local >= 0 && blocks + sink + local >= 1 && blocks + sink + local <= 65536,
              "1..65536 selected blocks");
    MDX_CHECK(aligned(ksum, 16) && s_head_stride % 8 == 0 && s_page_stride % 8 == 0 && s_head_stride >= 0 && s_page_stride >= D,
              "mean keys: 16-byte aligned rows");
    PagedArgs a{};
    const int rc = fill(a, q, q_seq_stride, q_row_stride, q_head_stride, key, k_head_stride, k_page_stride, k_row_stride, value,
                        v_head_stride, v_page_stride, v_row_stride, dtype, table, table_stride, length, mask, out, B, S, H, Hk, D, P,
                        T, W, scale);
    if (rc != MDX_OK) return rc;
    const int64_t most = blocks + sink + local, units = B * S * Hk;
    MDX_CHECK(H / Hk <= 64, "at most 64 query heads per kv head");
    MDX_CHECK(W <= 65536, "at most 65536 pages a sequence");
    MDX_CHECK(B * Hk <= 65535 && units < (int64_t(1) << 24) && units * (((most < W ? most : W) + 1) * T + S) / STEP + 8 * units < MAX_LINE,
              "too many rows times tokens for one call");
    const size_t need = mdx_attn_blocks_workspace(B, S, H, Hk, D, W, most);
    MDX_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= need, "workspace: %zu bytes, 16-byte aligned", need);
    a.spb = 1;
    a.units = int(S);
    a.most = int(most), a.sink = int(sink), a.local = int(local);
    a.ksum = static_cast<const uint16_t*>(ksum);
    a.sh = s_head_stride, a.sp = s_page_stride;
    a.sel = sel;
    a.info = static_cast<int4*>(workspace);
    a.part = reinterpret_cast<float*>(a.info + 2 * CUS);
    a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + base_bytes(a.G, D, Kind::SEL));
    a.page = reinterpret_cast<int32_t*>(a.keys + units * W);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (W > most) {  // (else every full page is selected)
        const dim3 grid(unsigned((W + 63) / 64), unsigned((S + SCORE_ROWS - 1) / SCORE_ROWS), unsigned(B * Hk));
        if (dtype == MDX_DT_BF16) {
            if (D == 64) hipLaunchKernelGGL((block_score_kernel<Bf16, 64>), grid, dim3(256), 0, st, a);
            else if (D == 128) hipLaunchKernelGGL((block_score_kernel<Bf16, 128>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((block_score_kernel<Bf16, 256>), grid, dim3(256), 0, st, a);
        } else {
            if (D == 64) hipLaunchKernelGGL((block_score_kernel<Fp16, 64>), grid, dim3(256), 0, st, a);
            else if (D == 128) hipLaunchKernelGGL((block_score_kernel<Fp16, 128>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((block_score_kernel<Fp16, 256>), grid, dim3(256), 0, st, a);
        }
        MDX_LAUNCHED();
    }
    // (keys in registers: the smallest form that holds a row's. A call at 1000 pages: 20.3 us, 21.7 by 256 threads of four keys,
    // 23.6 with the third form, 42.4 with the fourth; at 4000: 22.8, 24.1 by 512 threads of eight, 26.1, 46.4; at 16000: 34.6
    // with the third form and 62.5 with the fourth)
    if (W <= 1024) hipLaunchKernelGGL((block_select_kernel<512, 2>), dim3(unsigned(units)), dim3(512), 0, st, a);
    else if (W <= 4096) hipLaunchKernelGGL((block_select_kernel<1024, 4>), dim3(unsigned(units)), dim3(1024), 0, st, a);
    else if (W <= 16384) hipLaunchKernelGGL((block_select_kernel<1024, 16>), dim3(unsigned(units)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((block_select_kernel<1024, 64>), dim3(unsigned(units)), dim3(1024), 0, st, a);
    MDX_LAUNCHED();
    return launch_any<Kind::SEL>(a, int(D), dtype, st);
}
