// Verification of drafted tokens against the target's probabilities (mdx_verify_drafts).
//
// p_r = softmax(target row r / T), q_r = softmax(draft row r / T) of sequence b. From row 0 on:
//   with q (a chain): row r + 1, token x, is accepted if u_r q_r(x) < p_r(x); the first refusal draws the answer from
//     max(p_r - q_r, 0), which makes the answers distributed as the target's own;
//   without (drafts that are no samples, trees): the children of a row split [0, 1) by their p in row order, u_r takes one of
//     them or none; then the answer is drawn from p_r without them.
// The draw: the lowest index whose cumulative weight passes u_R of the whole.
//
// All of it in 64 bits: a drawn token is a whole number that changes where u falls between two sums, and at a vocabulary of 150
// thousand 32-bit sums (1e-7 of the whole) would move one draw in thirty across a border; 64-bit ones (1e-13) one in 1e8.
//
// Three launches. verify_rows_kernel: a work-group per slice of a row (16384 logits, fewer where there are few) sums their
// exponentials. verify_walk_kernel: a work-group per piece of a sequence's vocabulary joins the rows' sums, walks the tree (every
// work-group of a sequence alike, from LDS) and sums the weights of its piece of the row that answers. verify_draw_kernel: a
// work-group per sequence finds the run of 512 that the draw falls in and the token in it. (The last work-group of the second
// launch can not do that cheaply: a release to the other XCDs' caches by each of 600 cost 30 us.)
//
// What bounds it: many rows the exponentials, 14 vector instructions each, eight of them float64 (7 rows of 32 sequences and their
// drafts over 151936: 37 us for 126 MB, 25 at the rate of a large copy; with 20 instructions 51), then the walk and the draw, 18
// and 10 us, chains of dependent loads; one short chain those alone (16 us a call).
// Exponentials: 2^(a / 128) = table[k % 128] 2^(k / 128) poly(a - k), k = rint(a): a table of 1 KiB in LDS, a polynomial of degree 3
// through the Chebyshev points of [-1/2, 1/2] (2.8e-13 relative); x / T as it stands, without a maximum, as long as none is past
// 2^900 (then the row is read again less its largest).
//
// Reference: the walk's role is csrc/mtp_loop.sycl:86-196's accept (which compares with one sampled token per row).
#include "mdx_common.hpp"

namespace mdx {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_ROWS = 64;
constexpr int NT = 256;
constexpr int slice_of(int each) { return NT * each * 8; }  // logits of a work-group of `each` pieces of 8 per thread

constexpr int SUB = 512;  // logits that a wave holds side by side (8 per lane): the draw's runs

struct Part {  // of a slice of a row
    double sum;  // sum of exp((x - ref) / T)
    float ref;   // 0 where no x / T is far from it, else the largest x; -inf: nothing there
    int32_t at;  // T = 0: the lowest index of the largest x, which ref is
};

struct Answer {  // the row that answers
    double zp, zq;  // 1 / sum of the target's and the draft's row
    float rp, rq;   // their references
    int row;
    int refused;  // a token of q was refused there: max(p - q, 0)
};

struct VerifyArgs {
    const void* logits;  // [B, R, V], strides lb, lr
    int64_t lb, lr;
    const void* draft;   // [B, R - 1, V], strides db, dr; null: none
    int64_t db, dr;
    const int64_t* tokens;   // [B, R]
    const int32_t* parent;   // [B, R] or null (a chain)
    const double* uniform;   // [B, R + 1]
    const float* heat;       // [B] or null
    float one_heat;
    int32_t* count;  // [B]
    int32_t* path;   // [B, R]
    int64_t* next;   // [B]
    Part* part;      // [B][2 R - 1 or R][slices]
    double* sums;    // [B][runs of SUB logits]
    struct Answer* answer;  // [B]
    int B, R, V, rows;   // rows: of a sequence, the draft's behind the target's
    int slices, pieces;  // of a row: work-groups of the first launch, of the second
};

// ---- exponentials -----------------------------------------------------------------------------------------
constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: the low word of MAGIC + x is rint(x)
constexpr int STEPS = 128;                      // of an octave
constexpr float FAR = 900.f * STEPS;          // references past which 2^(a / STEPS) is taken less the largest a
constexpr double LEAST = -1020.0 * STEPS;     // a weight that counts as none

__device__ const double POWERS[STEPS] = {  // 2^(j / STEPS)
    0x1.0000000000000p+0, 0x1.0163da9fb3335p+0, 0x1.02c9a3e778061p+0, 0x1.04315e86e7f85p+0, 0x1.059b0d3158574p+0,
    0x1.0706b29ddf6dep+0, 0x1.0874518759bc8p+0, 0x1.09e3ecac6f383p+0, 0x1.0b5586cf9890fp+0, 0x1.0cc922b7247f7p+0,
    0x1.0e3ec32d3d1a2p+0, 0x1.0fb66affed31bp+0, 0x1.11301d0125b51p+0, 0x1.12abdc06c31ccp+0, 0x1.1429aaea92de0p+0,
    0x1.15a98c8a58e51p+0, 0x1.172b83c7d517bp+0, 0x1.18af9388c8deap+0, 0x1.1a35beb6fcb75p+0, 0x1.1bbe084045cd4p+0,
    0x1.1d4873168b9aap+0, 0x1.1ed5022fcd91dp+0, 0x1.2063b88628cd6p+0, 0x1.21f49917ddc96p+0, 0x1.2387a6e756238p+0,
    0x1.251ce4fb2a63fp+0, 0x1.26b4565e27cddp+0, 0x1.284dfe1f56381p+0, 0x1.29e9df51fdee1p+0, 0x1.2b87fd0dad990p+0,
    0x1.2d285a6e4030bp+0, 0x1.2ecafa93e2f56p+0, 0x1.306fe0a31b715p+0, 0x1.32170fc4cd831p+0, 0x1.33c08b26416ffp+0,
    0x1.356c55f929ff1p+0, 0x1.371a7373aa9cbp+0, 0x1.38cae6d05d866p+0, 0x1.3a7db34e59ff7p+0, 0x1.3c32dc313a8e5p+0,
    0x1.3dea64c123422p+0, 0x1.3fa4504ac801cp+0, 0x1.4160a21f72e2ap+0, 0x1.431f5d950a897p+0, 0x1.44e086061892dp+0,
    0x1.46a41ed1d0057p+0, 0x1.486a2b5c13cd0p+0, 0x1.4a32af0d7d3dep+0, 0x1.4bfdad5362a27p+0, 0x1.4dcb299fddd0dp+0,
    0x1.4f9b2769d2ca7p+0, 0x1.516daa2cf6642p+0, 0x1.5342b569d4f82p+0, 0x1.551a4ca5d920fp+0, 0x1.56f4736b527dap+0,
    0x1.58d12d497c7fdp+0, 0x1.5ab07dd485429p+0, 0x1.5c9268a5946b7p+0, 0x1.5e76f15ad2148p+0, 0x1.605e1b976dc09p+0,
    0x1.6247eb03a5585p+0, 0x1.6434634ccc320p+0, 0x1.6623882552225p+0, 0x1.68155d44ca973p+0, 0x1.6a09e667f3bcdp+0,
    0x1.6c012750bdabfp+0, 0x1.6dfb23c651a2fp+0, 0x1.6ff7df9519484p+0, 0x1.71f75e8ec5f74p+0, 0x1.73f9a48a58174p+0,
    0x1.75feb564267c9p+0, 0x1.780694fde5d3fp+0, 0x1.7a11473eb0187p+0, 0x1.7c1ed0130c132p+0, 0x1.7e2f336cf4e62p+0,
    0x1.80427543e1a12p+0, 0x1.82589994cce13p+0, 0x1.8471a4623c7adp+0, 0x1.868d99b4492edp+0, 0x1.88ac7d98a6699p+0,
    0x1.8ace5422aa0dbp+0, 0x1.8cf3216b5448cp+0, 0x1.8f1ae99157736p+0, 0x1.9145b0b91ffc6p+0, 0x1.93737b0cdc5e5p+0,
    0x1.95a44cbc8520fp+0, 0x1.97d829fde4e50p+0, 0x1.9a0f170ca07bap+0, 0x1.9c49182a3f090p+0, 0x1.9e86319e32323p+0,
    0x1.a0c667b5de565p+0, 0x1.a309bec4a2d33p+0, 0x1.a5503b23e255dp+0, 0x1.a799e1330b358p+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ac36bbfd3f37ap+0, 0x1.ae89f995ad3adp+0, 0x1.b0e07298db666p+0, 0x1.b33a2b84f15fbp+0, 0x1.b59728de5593ap+0,
    0x1.b7f76f2fb5e47p+0, 0x1.ba5b030a1064ap+0, 0x1.bcc1e904bc1d2p+0, 0x1.bf2c25bd71e09p+0, 0x1.c199bdd85529cp+0,
    0x1.c40ab5fffd07ap+0, 0x1.c67f12e57d14bp+0, 0x1.c8f6d9406e7b5p+0, 0x1.cb720dcef9069p+0, 0x1.cdf0b555dc3fap+0,
    0x1.d072d4a07897cp+0, 0x1.d2f87080d89f2p+0, 0x1.d5818dcfba487p+0, 0x1.d80e316c98398p+0, 0x1.da9e603db3285p+0,
    0x1.dd321f301b460p+0, 0x1.dfc97337b9b5fp+0, 0x1.e264614f5a129p+0, 0x1.e502ee78b3ff6p+0, 0x1.e7a51fbc74c83p+0,
    0x1.ea4afa2a490dap+0, 0x1.ecf482d8e67f1p+0, 0x1.efa1bee615a27p+0, 0x1.f252b376bba97p+0, 0x1.f50765b6e4540p+0,
    0x1.f7bfdad9cbe14p+0, 0x1.fa7c1819e90d8p+0, 0x1.fd3c22b8f71f1p+0};
// 2^(j / STEPS), the exponent less j << 13 in the high word: k << 13 added gives 2^(k / STEPS) for k % STEPS = j
__device__ __forceinline__ void fill_table(double* tab) {  // (the caller's barrier follows)
    const int j = threadIdx.x;
    if (j < STEPS) {
        const double v = POWERS[j];
        tab[j] = __hiloint2double(__double2hiint(v) - (j << 13), __double2loint(v));
    }
}
__device__ __forceinline__ double poly(double f) {
    double p = __builtin_fma(f, 0x1.c6b0985c8a1bcp-26, 0x1.ebfbf3aad80f5p-17);
    p = __builtin_fma(p, f, 0x1.62e42fefa3892p-8);
    return __builtin_fma(p, f, 0x1.ffffffffff627p-1);
}
__device__ __forceinline__ double power(int k, const double* tab) {
    const double v = tab[k & (STEPS - 1)];
    return __hiloint2double(__double2hiint(v) + (k << 13), __double2loint(v));
}
// 2^(a / STEPS); below 2^-1020 (NaN too) that
__device__ __forceinline__ double exp2_steps(double a, const double* tab) {
    a = __builtin_fmax(a, LEAST);
    const double t = a + MAGIC;
    return poly(a - (t - MAGIC)) * power(__double2loint(t), tab);
}
// sum + 2^(x c / STEPS), |x c| at most 1020 STEPS: eight float64 instructions
__device__ __forceinline__ double add_exp(double sum, float x, double c, const double* tab) {
    const double d = double(x), t = __builtin_fma(d, c, MAGIC);
    return __builtin_fma(poly(__builtin_fma(d, c, MAGIC - t)), power(__double2loint(t), tab), sum);
}
// STEPS log2(e) / T, 0 for the largest logit alone (T past 1e30 counts as that: a logit of -inf stays one that has nothing)
__device__ __forceinline__ double rate_of(const VerifyArgs& a, int b) {
    const float t = a.heat ? a.heat[b] : a.one_heat;
    return t > 0.f ? __builtin_fmax(STEPS * 1.4426950408889634074 / double(t), STEPS * 1.44e-30) : 0.0;
}
__device__ __forceinline__ bool greedy(const VerifyArgs& a, int b) { return !((a.heat ? a.heat[b] : a.one_heat) > 0.f); }

// ---- logits -----------------------------------------------------------------------------------------------
struct Bf {
    typedef uint16_t type;
    static constexpr uint16_t NONE = 0xFF80;  // -inf
    static __device__ __forceinline__ float f32(uint16_t x) { return bf2f(x); }
};
struct Hf {
    typedef uint16_t type;
    static constexpr uint16_t NONE = 0xFC00;
    static __device__ __forceinline__ float f32(uint16_t x) { return fp16_to_f32(x); }
};
struct Ff {
    typedef float type;
    static constexpr float NONE = -INFINITY;
    static __device__ __forceinline__ float f32(float x) { return x; }
};
template <class E>
__device__ __forceinline__ const typename E::type* row_of(const VerifyArgs& a, int b, int r) {  // r >= R: the draft's row r - R
    typedef typename E::type T;
    return r < a.R ? static_cast<const T*>(a.logits) + b * a.lb + r * a.lr : static_cast<const T*>(a.draft) + b * a.db + (r - a.R) * a.dr;
}
// elements between the 16-byte boundary before the row and the row
template <class E>
__device__ __forceinline__ int shift_of(const typename E::type* row) {
    return int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::type));
}
// a NaN counts as nothing, an infinity as the largest finite number
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f); }

// Eight logits as they stand in memory.
template <class E>
struct Piece {
    static constexpr int W = sizeof(typename E::type) * 8 / 16;
    u32x4 v[W];
    __device__ __forceinline__ float operator[](int k) const {
        if constexpr (W == 1) return E::f32(uint16_t(v[0][k / 2] >> (16 * (k & 1))));
        else return __uint_as_float(v[k / 4][k & 3]);
    }
};
// The eight from e on, -inf outside of the row; `even`: e is at a 16-byte boundary.
template <class E>
__device__ __forceinline__ Piece<E> piece_at(const typename E::type* row, int V, int e, bool even) {
    typedef typename E::type T;
    Piece<E> p;
    if (even && e >= 0 && e + 8 <= V) {
#pragma unroll
        for (int j = 0; j < Piece<E>::W; ++j) p.v[j] = *reinterpret_cast<const u32x4*>(row + e + j * (16 / int(sizeof(T))));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            T x = E::NONE;
            if (e + k >= 0 && e + k < V) x = row[e + k];
            if constexpr (Piece<E>::W == 1) p.v[0][k / 2] = k & 1 ? p.v[0][k / 2] | (unsigned(x) << 16) : unsigned(x);
            else p.v[k / 4][k & 3] = __float_as_uint(x);
        }
    }
    return p;
}
// This thread's piece i of slice `slice` begins at logit at0(i).
template <int EACH>
__device__ __forceinline__ int at0(int slice, int i, int shift) {
    return (slice * (NT * EACH) + i * NT + int(threadIdx.x)) * 8 - shift;
}

// ---- sums over a wave -------------------------------------------------------------------------------------------
// (the lanes across by DPP and lane exchanges: the LDS crossbar's steps are six times as long)
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double across(double v) {  // 0 where there is no such lane
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ double wave_sum(double v) {  // in every lane
    v += across<0x128>(v);  // lane ^ 8 of the 16, ^ 7, ^ 3, ^ 1
    v += across<0x141>(v);
    v += across<0x1B>(v);
    v += across<0xB1>(v);
    const auto l16 = __builtin_amdgcn_permlane16_swap(unsigned(__double2loint(v)), unsigned(__double2loint(v)), false, false);
    const auto h16 = __builtin_amdgcn_permlane16_swap(unsigned(__double2hiint(v)), unsigned(__double2hiint(v)), false, false);
    v = __hiloint2double(int(h16[0]), int(l16[0])) + __hiloint2double(int(h16[1]), int(l16[1]));
    const auto l32 = __builtin_amdgcn_permlane32_swap(unsigned(__double2loint(v)), unsigned(__double2loint(v)), false, false);
    const auto h32 = __builtin_amdgcn_permlane32_swap(unsigned(__double2hiint(v)), unsigned(__double2hiint(v)), false, false);
    return __hiloint2double(int(h32[0]), int(l32[0])) + __hiloint2double(int(h32[1]), int(l32[1]));
}
__device__ __forceinline__ double wave_scan(double v) {  // inclusive, in lane order
    v += across<0x111>(v);  // the lane 1, 2, 4, 8 ahead in the row of 16
    v += across<0x112>(v);
    v += across<0x114>(v);
    v += across<0x118>(v);
    v += across<0x142, 0xA>(v);  // row 0's last lane to row 1, 2's to 3; then row 1's to 2 and 3
    v += across<0x143, 0xC>(v);
    return v;
}

// ---- the rows' sums ---------------------------------------------------------------------------------------------
// the larger of a and the magnitudes of b and c (a NaN counts as nothing)
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// A slice of a row. The sums are taken as if no x / T were far from 0, nor -inf; where one is, or T is 0, the slice is read again.
template <class E, int EACH>
__global__ __launch_bounds__(NT) void verify_rows_kernel(VerifyArgs a) {
    __shared__ double tab[STEPS], sum_w[NT / 64];
    __shared__ float ref_w[NT / 64];
    __shared__ int at_w[NT / 64];
    const int slice = int(blockIdx.x % unsigned(a.slices)), r = int(blockIdx.x / unsigned(a.slices)) % a.rows,
              b = int(blockIdx.x / unsigned(a.slices)) / a.rows;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const typename E::type* row = row_of<E>(a, b, r);
    const int shift = shift_of<E>(row);
    Piece<E> x[EACH];
    const int first = slice * slice_of(EACH) + w * SUB - shift;  // the wave's first logit; its pieces are 2048 apart
    if (first >= 0 && first + (EACH - 1) * NT * 8 + SUB <= a.V) {  // (uniform)
        const typename E::type* from = row + first + lane * 8;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int j = 0; j < Piece<E>::W; ++j) x[i].v[j] = *reinterpret_cast<const u32x4*>(from + i * NT * 8 + j * (16 / int(sizeof(*from))));
    } else {
#pragma unroll
        for (int i = 0; i < EACH; ++i) x[i] = piece_at<E>(row, a.V, at0<EACH>(slice, i, shift), true);
    }
    fill_table(tab);
    const double c = rate_of(a, b);
    __syncthreads();  // (the table)
    double s0 = 0, s1 = 0;
    float top = -1.f, ref = 0.f;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = first + i * NT * 8;
        if (e >= a.V) break;  // (uniform)
        if (e >= 0 && e + SUB <= a.V) {
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const float x0 = x[i][k], x1 = x[i][k + 1];
                top = max3_abs(top, x0, x1);
                s0 = add_exp(s0, x0, c, tab);
                s1 = add_exp(s1, x1, c, tab);
            }
        } else {  // (an end of the row: what is -inf counts as 2^-1020)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float y = x[i][k];
                if (y > -INFINITY) top = fmaxf(top, __builtin_fabsf(y));
                s0 += exp2_steps(double(y) * c, tab);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (eight at a time are enough in flight: more cost registers, and waves)
    }
    double s = s0 + s1;
    // (a NaN makes the sum one; a lane past the row's end has top -1)
    const bool near = c > 0.0 && double(top) * c < FAR && s == s;
    if (__builtin_amdgcn_ballot_w64(!near) != 0 || __builtin_amdgcn_ballot_w64(top >= 0.f) == 0) {  // (uniform in the wave)
        // once more: the largest, and whether a reference of 0 will do with the others raised to weights of 2^-1020
        ref = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < EACH; ++i) {
            const int e = at0<EACH>(slice, i, shift);
            const Piece<E> y = piece_at<E>(row, a.V, e, true);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float z = clean(y[k]);
                if (z > ref) at = e + k;
                ref = fmaxf(ref, z);
            }
        }
        const float mine = ref;
        ref = wave_max(ref);
        if (mine < ref || ref == -INFINITY || c > 0.0) at = 0x7FFFFFFF;
        for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d, 64));
        s = 0;
        if (ref > -INFINITY && c > 0.0) {
            const bool zero = __builtin_fabs(double(ref) * c) < FAR;
            const double less = zero ? 0.0 : double(ref);
#pragma unroll 1
            for (int i = 0; i < EACH; ++i) {
                const Piece<E> y = piece_at<E>(row, a.V, at0<EACH>(slice, i, shift), true);
#pragma unroll
                for (int k = 0; k < 8; ++k) s += exp2_steps((double(clean(y[k])) - less) * c, tab);
            }
            if (zero) ref = 0.f;
        }
    }
    s = wave_sum(s);
    if (lane == 0) {
        sum_w[w] = s;
        ref_w[w] = ref;
        at_w[w] = at;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    float all = ref_w[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) all = fmaxf(all, ref_w[i]);
    double sum = 0;
    int lowest = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        if (ref_w[i] == -INFINITY) continue;
        sum += ref_w[i] == all ? sum_w[i] : sum_w[i] * exp2_steps((double(ref_w[i]) - double(all)) * c, tab);
        if (ref_w[i] == all) lowest = min(lowest, at_w[i]);
    }
    a.part[(int64_t(b) * a.rows + r) * a.slices + slice] = Part{sum, all, lowest};
}

// ---- the walk and the draw ------------------------------------------------------------------------------------
// a logit's probability in a row of reference ref and 1 / sum z: none for -inf and what lies 2^1020 below the reference
struct Soft {
    double c, z, ref;
    float cut;
    bool none;
    __device__ __forceinline__ Soft(double c_, double z_, float r) : c(c_), z(z_), ref(r), none(!(r > -INFINITY)) {
        cut = fmaxf(-3.402823466e38f, float(ref + LEAST / c));
    }
    __device__ __forceinline__ double of(float x, const double* tab) const {
        const float y = fmaxf(x, cut);
        const double e = ref == 0.0 ? add_exp(0.0, y, c, tab) : exp2_steps((double(fminf(y, 3.402823466e38f)) - ref) * c, tab);
        return x >= cut && !none ? e * z : 0.0;
    }
};

// The weights of the eight logits from e0 on (8 lanes apart in a wave) of the row that answers. up, tok (LDS): the rows' parents
// and tokens, -1: none.
template <class E, int N>
__device__ __forceinline__ void weights(const VerifyArgs& a, int b, const Answer& w, double c, const int (&e0)[N], bool rest, const int* up,
                                        const int64_t* tok, const double* tab, double (&wt)[N][8]) {
    const typename E::type *pr = row_of<E>(a, b, w.row), *qr = rest ? row_of<E>(a, b, a.R + w.row) : pr;
    const bool alike = shift_of<E>(pr) == shift_of<E>(qr);  // (to the 16-byte boundaries)
    Piece<E> x[N], y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = piece_at<E>(pr, a.V, e0[i], true);
    if (rest)  // (uniform)
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_at<E>(qr, a.V, e0[i], alike);
    const Soft p(c, w.zp, w.rp), q(c, w.zq, w.rq);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            wt[i][k] = p.of(x[i][k], tab);
            if (rest) wt[i][k] = __builtin_fmax(wt[i][k] - q.of(y[i][k], tab), 0.0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (a.draft) return;
    for (int s = w.row + 1; s < a.R; ++s) {  // the children that were tried
        if (up[s] != w.row) continue;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (int(tok[s]) == e0[i] + k) wt[i][k] = 0.0;
    }
}
// row t's token and parent (thread t): what can be reached
__device__ __forceinline__ void row_at(const VerifyArgs& a, int b, int t, int64_t& x, int& parent) {
    x = a.tokens[int64_t(b) * a.R + t];
    parent = t == 0 ? -1 : a.parent ? a.parent[int64_t(b) * a.R + t] : t - 1;
    if (!(t > 0 && x >= 0 && x < a.V && parent >= 0 && parent < t)) x = parent = -1;
}

template <class E, int EACH>
__global__ __launch_bounds__(NT) void verify_walk_kernel(VerifyArgs a) {
    __shared__ double tab[STEPS], z[2 * MAX_ROWS], share[MAX_ROWS];
    __shared__ float ref[2 * MAX_ROWS];
    __shared__ int best[2 * MAX_ROWS], up[MAX_ROWS], took[MAX_ROWS], line[MAX_ROWS], pick[2];
    __shared__ int64_t tok[MAX_ROWS];
    const int slice = int(blockIdx.x % unsigned(a.pieces)), b = int(blockIdx.x / unsigned(a.pieces));
    const int t = threadIdx.x;
    const double c = rate_of(a, b);
    const bool cold = greedy(a, b);
    // thread r: row r's token, its parent, and the token's logits there
    int64_t x = -1;
    int parent = -1;
    float own_p = -INFINITY, own_q = -INFINITY;
    double own_u = 0;
    if (t < a.R) {
        row_at(a, b, t, x, parent);
        tok[t] = x;
        up[t] = parent;
        took[t] = -1;
        if (parent >= 0) {
            own_p = E::f32(row_of<E>(a, b, parent)[x]);
            if (a.draft) own_q = E::f32(row_of<E>(a, b, a.R + parent)[x]);
            own_u = a.uniform[int64_t(b) * (a.R + 1) + parent];
        }
    }
    fill_table(tab);
    __syncthreads();
    // 16 lanes a row: its reference and sum out of the slices', four of them in flight
    for (int r = t >> 4; r < a.rows; r += NT / 16) {
        const Part* part = a.part + (int64_t(b) * a.rows + r) * a.slices;
        float m = -INFINITY;
        double s = 0;
        int at = 0x7FFFFFFF;
        for (int i0 = t & 15; i0 < a.slices; i0 += 64) {
            Part p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = part[min(i0 + 16 * j, a.slices - 1)];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i0 + 16 * j >= a.slices || p[j].ref == -INFINITY) continue;
                if (p[j].ref == m) {
                    s += p[j].sum;
                    at = min(at, p[j].at);
                } else if (p[j].ref > m) {
                    s = (m == -INFINITY ? 0.0 : s * exp2_steps((double(m) - double(p[j].ref)) * c, tab)) + p[j].sum;
                    m = p[j].ref;
                    at = p[j].at;
                } else {
                    s += p[j].sum * exp2_steps((double(p[j].ref) - double(m)) * c, tab);
                }
            }
        }
        float all = m;
        for (int d = 8; d; d >>= 1) all = fmaxf(all, __shfl_xor(all, d, 64));
        if (m != all) s = m == -INFINITY ? 0.0 : s * exp2_steps((double(m) - double(all)) * c, tab);
        at = m == all ? at : 0x7FFFFFFF;
        for (int d = 8; d; d >>= 1) {
            s += __shfl_xor(s, d, 64);
            at = min(at, __shfl_xor(at, d, 64));
        }
        if ((t & 15) == 0) {
            ref[r] = all;
            z[r] = all == -INFINITY ? 0.0 : 1.0 / s;
            best[r] = all == -INFINITY ? -1 : at;
        }
    }
    __syncthreads();
    // probability of this thread's token in its parent's row (r >= R: the draft's)
    auto prob = [&](int r, float l) -> double { return cold ? (x == best[r] ? 1.0 : 0.0) : Soft(c, z[r], ref[r]).of(l, tab); };
    if (parent >= 0) {
        bool again = false;  // (a token that a sibling ahead has tried)
        for (int s = 1; s < t && !a.draft; ++s) again = again || (up[s] == parent && tok[s] == x);
        share[t] = again ? 0.0 : prob(parent, own_p);
    }
    __syncthreads();
    if (parent >= 0) {
        bool ok;
        if (a.draft) {
            ok = own_u * prob(a.R + parent, own_q) < share[t];
        } else {  // the siblings ahead have [0, from)
            double from = 0;
            for (int s = 1; s < t; ++s) from += up[s] == parent ? share[s] : 0.0;
            ok = own_u < from + share[t] && !(own_u < from);
        }
        if (ok) took[parent] = t;  // (one child at most: their parts of [0, 1) do not meet)
    }
    __syncthreads();
    if (t == 0) {
        int n = 0, at = 0;
        line[n++] = 0;
        while (took[at] >= 0) line[n++] = at = took[at];  // (a child's row is behind its parent's)
        pick[0] = at;
        pick[1] = n;
    }
    __syncthreads();
    const int row = pick[0], n = pick[1];
    const bool refused = a.draft && row + 1 < a.R && up[row + 1] == row;
    const Answer w{z[row], refused ? z[a.R + row] : 0.0, ref[row], refused ? ref[a.R + row] : 0.f, row, refused};
    if (slice == 0) {
        if (t < a.R) a.path[int64_t(b) * a.R + t] = t < n ? line[t] : -1;
        if (t == 0) {
            a.count[b] = n;
            a.answer[b] = w;
            if (cold) a.next[b] = best[row];
        }
    }
    if (cold) return;  // (uniform)
    // the sum of every wave's runs of SUB logits
    double wt[EACH][8];
    int e0[EACH];
    const int shift = shift_of<E>(row_of<E>(a, b, row));
#pragma unroll
    for (int i = 0; i < EACH; ++i) e0[i] = at0<EACH>(slice, i, shift);
    weights<E, EACH>(a, b, w, c, e0, refused, up, tok, tab, wt);
    double* sums = a.sums + (int64_t(b) * a.pieces + slice) * (EACH * (NT / 64)) + (t >> 6);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        double s = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += wt[i][k];
        s = wave_sum(s);
        if ((t & 63) == 0) sums[i * (NT / 64)] = s;
    }
}

constexpr int DT = 512;  // threads of the draw: all runs of a vocabulary of 262144 at once
template <class E>
__global__ __launch_bounds__(DT) void verify_draw_kernel(VerifyArgs a, int runs) {
    __shared__ double tab[STEPS], tmp[DT / 64], aim;
    __shared__ int up[MAX_ROWS], pick[2];
    __shared__ int64_t tok[MAX_ROWS];
    const int t = threadIdx.x, b = int(blockIdx.x), lane = t & 63;
    const double c = rate_of(a, b);
    if (greedy(a, b)) return;  // (uniform: the walk has written the answer)
    double* sums = a.sums + int64_t(b) * runs;
    const double mine = t < runs ? sums[t] : 0.0;
    const Answer w = a.answer[b];
    const double u = a.uniform[int64_t(b) * (a.R + 1) + a.R];
    if (t < a.R) row_at(a, b, t, tok[t], up[t]);
    fill_table(tab);
    const int shift = shift_of<E>(row_of<E>(a, b, w.row));
    // inclusive sum over the work-group's threads in order, and the total (every thread calls it)
    auto block_scan = [&](double v, double& total) {
        v = wave_scan(v);
        __syncthreads();  // (tmp may be in use by the call before)
        if (lane == 63) tmp[t >> 6] = v;
        __syncthreads();
        double before = 0;
        total = 0;
#pragma unroll
        for (int i = 0; i < DT / 64; ++i) {
            before += i < (t >> 6) ? tmp[i] : 0.0;
            total += tmp[i];
        }
        return v + before;
    };
    // The run that the draw falls in: the first whose sum, with those ahead, passes u of all (the last that has any); the aim
    // within it.
    auto find = [&](double s) {
        double total, part;
        double upto = block_scan(s, total);
        const bool once = runs <= DT;
        if (!once) {
            for (int i0 = DT; i0 < runs; i0 += DT) {
                block_scan(i0 + t < runs ? sums[i0 + t] : 0.0, part);
                total += part;
            }
        }
        const double to = u * total;
        if (t == 0) pick[0] = 0x7FFFFFFF, pick[1] = -1;
        double before = 0;
        for (int i0 = 0; i0 < runs; i0 += DT) {
            if (!once) {
                s = i0 + t < runs ? sums[i0 + t] : 0.0;
                upto = before + block_scan(s, part);
                before += part;
            }
            __syncthreads();
            if (s > 0) {
                atomicMax(&pick[1], i0 + t);
                if (upto > to) atomicMin(&pick[0], i0 + t);
            }
            __syncthreads();
            const bool passed = pick[0] < runs;
            if ((passed ? pick[0] : pick[1]) == i0 + t) aim = to - (upto - s);  // (of the last with any as long as none passes)
            if (passed) break;  // (uniform)
        }
        __syncthreads();
        return pick[0] < runs ? pick[0] : pick[1];
    };
    bool rest = w.refused;
    double wt[1][8];
    int from = find(mine);
    if (from < 0 && rest) {  // (uniform) nothing is left of p - q: the answer is p's
        rest = false;
        for (int i = t >> 6; i < runs; i += DT / 64) {
            const int e0[1] = {i * SUB + lane * 8 - shift};
            weights<E, 1>(a, b, w, c, e0, false, up, tok, tab, wt);
            double s = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += wt[0][k];
            s = wave_sum(s);
            if (lane == 0) sums[i] = s;
        }
        __syncthreads();
        from = find(t < runs ? sums[t] : 0.0);
    }
    if (t >= 64) return;
    if (from < 0) {
        if (t == 0) a.next[b] = -1;
        return;
    }
    // ---- and the token in it, by the first wave
    const int e0[1] = {from * SUB + lane * 8 - shift};
    weights<E, 1>(a, b, w, c, e0, rest, up, tok, tab, wt);
    double s = 0;
    int last = -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        s += wt[0][k];
        if (wt[0][k] > 0) last = k;
    }
    const double upto = wave_scan(s), to = aim;
    const uint64_t past = __builtin_amdgcn_ballot_w64(last >= 0 && upto > to), any = __builtin_amdgcn_ballot_w64(last >= 0);
    if (any == 0) return;  // (not reached: the run's sum is not zero)
    if (lane != (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any))) return;
    double run = upto - s;
    int at = -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        run += wt[0][k];
        if (at < 0 && wt[0][k] > 0 && run > to) at = k;
    }
    a.next[b] = e0[0] + (at < 0 || !past ? last : at);  // (the last with a weight, where rounding lets none pass)
}

template <class E, int ROWS, int WALK>
int launch(const VerifyArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((verify_rows_kernel<E, ROWS>), dim3(unsigned(int64_t(a.slices) * a.rows * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_walk_kernel<E, WALK>), dim3(unsigned(a.pieces * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_draw_kernel<E>), dim3(unsigned(a.B)), dim3(DT), 0, st, a, a.pieces * WALK * (NT / 64));
    MDX_LAUNCHED();
    return MDX_OK;
}
template <class E>
int launch_any(const VerifyArgs& a, int rows, int walk, hipStream_t st) {
    if (rows == 8) return walk == 4 ? launch<E, 8, 4>(a, st) : launch<E, 8, 1>(a, st);
    if (rows == 4) return walk == 4 ? launch<E, 4, 4>(a, st) : launch<E, 4, 1>(a, st);
    return walk == 4 ? launch<E, 1, 4>(a, st) : launch<E, 1, 1>(a, st);
}

int64_t slices_of(int64_t V, int each) { return (V + 7 + slice_of(each) - 1) / slice_of(each); }
// Pieces of eight logits per thread: as many as leave work-groups enough (their exponentials are a chain of 2 us).
int rows_each(int64_t B, int64_t rows, int64_t V) { return B * rows * slices_of(V, 8) >= 2048 ? 8 : B * rows * slices_of(V, 4) >= 1024 ? 4 : 1; }
int walk_each(int64_t B, int64_t V) { return B * slices_of(V, 1) > 2048 ? 4 : 1; }
int64_t runs_of(int64_t B, int64_t V) { return slices_of(V, walk_each(B, V)) * walk_each(B, V) * (NT / 64); }  // (a multiple of 4)

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_verify_drafts_workspace(int64_t B, int64_t R, int64_t V, int32_t drafted) {
    if (B < 1 || B > 1024 || R < 1 || R > MAX_ROWS || V < 1 || V >= (int64_t(1) << 24)) return 0;
    const int64_t rows = drafted ? 2 * R - 1 : R, slices = slices_of(V, rows_each(B, rows, V));
    return size_t(B * rows * slices) * sizeof(Part) + size_t(B * runs_of(B, V)) * 8 + size_t(B) * sizeof(Answer);
}

extern "C" int mdx_verify_drafts(const void* logits, int64_t seq_stride, int64_t row_stride, const void* draft,
                                 int64_t draft_seq_stride, int64_t draft_row_stride, int32_t dtype, const int64_t* tokens,
                                 const int32_t* parent, const double* uniform, const float* temperatures, float temperature,
                                 int32_t* count, int32_t* path, int64_t* next, int64_t B, int64_t R, int64_t V, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    MDX_CHECK(logits && tokens && uniform && count && path && next, "null pointer");
    MDX_CHECK(dtype == MDX_DT_BF16 || dtype == MDX_DT_F16 || dtype == MDX_DT_F32, "bf16, fp16 or fp32 logits");
    MDX_CHECK(B >= 1 && B <= 1024 && R >= 1 && R <= MAX_ROWS && V >= 1 && V < (int64_t(1) << 24),
              "1..1024 sequences, 1..64 rows, a vocabulary under 2^24");
    MDX_CHECK(!(draft && parent), "drafts with probabilities: a chain (no parents)");
    const int64_t lim = int64_t(1) << 40;
    MDX_CHECK(seq_stride >= 0 && row_stride >= 0 && seq_stride < lim && row_stride < lim && draft_seq_stride >= 0 && draft_row_stride >= 0 &&
                  draft_seq_stride < lim && draft_row_stride < lim,
              "strides");
    MDX_CHECK(temperatures || (temperature >= 0.f && temperature < INFINITY), "a temperature of 0 or more, finite");
    const bool drafted = draft && R > 1;
    const size_t need = mdx_verify_drafts_workspace(B, R, V, drafted);
    MDX_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= need, "workspace: %zu bytes, 16-byte aligned", need);
    VerifyArgs a{};
    a.logits = logits;
    a.lb = seq_stride, a.lr = row_stride;
    a.draft = drafted ? draft : nullptr;
    a.db = draft_seq_stride, a.dr = draft_row_stride;
    a.tokens = tokens;
    a.parent = parent;
    a.uniform = uniform;
    a.heat = temperatures;
    a.one_heat = temperature;
    a.count = count;
    a.path = path;
    a.next = next;
    a.B = int(B), a.R = int(R), a.V = int(V), a.rows = int(drafted ? 2 * R - 1 : R);
    const int rows = rows_each(B, a.rows, V), walk = walk_each(B, V);
    a.slices = int(slices_of(V, rows)), a.pieces = int(slices_of(V, walk));
    MDX_CHECK(B * a.rows * a.slices < (int64_t(1) << 30), "too many rows times logits for one call");
    a.part = static_cast<Part*>(workspace);
    a.sums = reinterpret_cast<double*>(a.part + B * a.rows * a.slices);
    a.answer = reinterpret_cast<Answer*>(a.sums + B * runs_of(B, V));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MDX_DT_BF16) return launch_any<Bf>(a, rows, walk, st);
    if (dtype == MDX_DT_F16) return launch_any<Hf>(a, rows, walk, st);
    return launch_any<Ff>(a, rows, walk, st);
}
