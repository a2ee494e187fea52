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
// thousand 32-bit weights and sums (1e-7 of the whole) would move one draw in a hundred across a border. Here a weight is good to some 2e-15 and
// 3e-16 |x / T|, a border to half of that: at most one draw in 1e9.
//
// verify_rows_kernel: a work-group per slice of a row (16384 logits, fewer where there are few) sums their exponentials. Without q
// it leaves the sums of every run of 512 logits too, and verify_answer_kernel, a work-group per sequence, joins the rows' sums,
// walks the tree, finds the run that the draw falls in, and the token in it. With q the weights of the row that answers are known
// after the walk alone: verify_walk_kernel, a work-group per piece of a sequence's vocabulary, joins and walks (every work-group of
// a sequence alike, from LDS) and sums the weights of its piece; verify_draw_kernel, a work-group per sequence, draws. (The last
// work-group of the second launch can not do that cheaply: a release to the other XCDs' caches by each of 600 cost 30 us.)
//
// What bounds it: many rows the exponentials, 14 vector instructions each, eight of them float64 (7 rows of 32 sequences and their
// drafts over 151936: 37 us for 126 MB, 25 at the rate of a large copy; with 20 instructions 51), then the walk and the draw, 16
// and 5 us, chains of dependent loads; one short chain those alone (14 us a call). 8 rows of 16 trees: 16 us and 11.
// Exponentials: 2^(a / 512) = table[k % 512] 2^((k - k % 512) / 512) poly(a - k), k = rint(a): a table of 4 KiB in LDS, a polynomial
// of degree 3 through the Chebyshev points of [-1/2, 1/2] (1.1e-15 relative; the rows of 32 sequences take 37 us, 35 with a table of
// 128 and 2.8e-13, 37.6 with one of 1024 and 1.1e-16); x / T as it stands, without a maximum, as long as none is past 2^900 (then the
// row is read again less its largest).
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
    Part* run;       // without drafts [B][R][runs of SUB logits], `at` unused
    double* sums;    // with drafts [B][runs]
    struct Answer* answer;  // with drafts [B]
    int B, R, V, rows;   // rows: of a sequence, the draft's behind the target's
    int slices, pieces;  // of a row: work-groups of the first launch, of the second
};

// ---- exponentials -----------------------------------------------------------------------------------------
constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: the low word of MAGIC + x is rint(x)
constexpr int STEPS = 512;                    // of an octave
constexpr float FAR = 900.f * STEPS;          // references past which 2^(a / STEPS) is taken less the largest a
constexpr double LEAST = -1020.0 * STEPS;     // a weight that counts as none

constexpr int FINE = 32;
__device__ const double COARSE[STEPS / FINE] = {  // 2^(j FINE / STEPS)
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0, 0x1.306fe0a31b715p+0,
    0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0, 0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0,
    0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0, 0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0,
    0x1.ea4afa2a490dap+0};
__device__ const double POWERS[FINE] = {  // 2^(j / STEPS)
    0x1.0000000000000p+0, 0x1.0058c86da1c0ap+0, 0x1.00b1afa5abcbfp+0, 0x1.010ab5b2cbd11p+0, 0x1.0163da9fb3335p+0,
    0x1.01bd1e77170b4p+0, 0x1.02168143b0281p+0, 0x1.027003103b10ep+0, 0x1.02c9a3e778061p+0, 0x1.032363d42b027p+0,
    0x1.037d42e11bbccp+0, 0x1.03d7411915a8ap+0, 0x1.04315e86e7f85p+0, 0x1.048b9b35659d8p+0, 0x1.04e5f72f654b1p+0,
    0x1.0540727fc1762p+0, 0x1.059b0d3158574p+0, 0x1.05f5c74f0bec2p+0, 0x1.0650a0e3c1f89p+0, 0x1.06ab99fa6407cp+0,
    0x1.0706b29ddf6dep+0, 0x1.0761ead925493p+0, 0x1.07bd42b72a836p+0, 0x1.0818ba42e7d30p+0, 0x1.0874518759bc8p+0,
    0x1.08d0088f8093fp+0, 0x1.092bdf66607e0p+0, 0x1.0987d61701716p+0, 0x1.09e3ecac6f383p+0, 0x1.0a402331b9715p+0,
    0x1.0a9c79b1f3919p+0, 0x1.0af8f03834e52p+0};
// 2^(j / STEPS), the exponent less j << SHIFT in the high word: k << SHIFT added gives 2^(k / STEPS) for k % STEPS = j
constexpr int SHIFT = 20 - 9;
static_assert(STEPS << SHIFT == 1 << 20, "");
template <int THREADS>
__device__ __forceinline__ void fill_table(double* tab) {  // (the caller's barrier follows)
#pragma unroll
    for (int i = 0; i < STEPS; i += THREADS) {
        const int j = i + int(threadIdx.x);
        if (STEPS % THREADS != 0 && j >= STEPS) break;
        const double v = COARSE[j / FINE] * POWERS[j % FINE];
        tab[j] = __hiloint2double(__double2hiint(v) - (j << SHIFT), __double2loint(v));
    }
}
__device__ __forceinline__ double poly(double f) {
    double p = __builtin_fma(f, 0x1.c6b08e52035e3p-32, 0x1.ebfbe133587d2p-21);
    p = __builtin_fma(p, f, 0x1.62e42fefa39efp-10);
    return __builtin_fma(p, f, 0x1.ffffffffffff6p-1);
}
__device__ __forceinline__ double power(int k, const double* tab) {
    const double v = tab[k & (STEPS - 1)];
    return __hiloint2double(__double2hiint(v) + (k << SHIFT), __double2loint(v));
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
// a's sums over the rows of 16 lanes 2 i and 2 i + 1, in row 2 i, b's in row 2 i + 1
__device__ __forceinline__ double join16(double a, double b) {
    const auto l = __builtin_amdgcn_permlane16_swap(unsigned(__double2loint(a)), unsigned(__double2loint(b)), false, false);
    const auto h = __builtin_amdgcn_permlane16_swap(unsigned(__double2hiint(a)), unsigned(__double2hiint(b)), false, false);
    return __hiloint2double(int(h[0]), int(l[0])) + __hiloint2double(int(h[1]), int(l[1]));
}
// a's sums over the halves of the wave, in the lower one, b's in the upper one
__device__ __forceinline__ double join32(double a, double b) {
    const auto l = __builtin_amdgcn_permlane32_swap(unsigned(__double2loint(a)), unsigned(__double2loint(b)), false, false);
    const auto h = __builtin_amdgcn_permlane32_swap(unsigned(__double2hiint(a)), unsigned(__double2hiint(b)), false, false);
    return __hiloint2double(int(h[0]), int(l[0])) + __hiloint2double(int(h[1]), int(l[1]));
}
__device__ __forceinline__ double row_sum(double v) {  // over 16 lanes, in each of them
    v += across<0x128>(v);  // lane ^ 8 of the 16, ^ 7, ^ 3, ^ 1
    v += across<0x141>(v);
    v += across<0x1B>(v);
    v += across<0xB1>(v);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {  // in every lane
    v = row_sum(v);
    v = join16(v, v);
    return join32(v, v);
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
// RUNS: the sums of every run too, for the draw.
template <class E, int EACH, bool RUNS>
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
    fill_table<NT>(tab);
    const double c = rate_of(a, b);
    __syncthreads();  // (the table)
    // the wave's run i
    auto put = [&](int i, double sum, float from) {
        a.run[((int64_t(b) * a.R + r) * a.slices + slice) * (EACH * (NT / 64)) + i * (NT / 64) + w] = Part{sum, from, 0};
    };
    double s = 0, s0 = 0, s1 = 0, one = 0, two = 0;
    float top = -1.f, ref = 0.f;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = first + i * NT * 8;
        if (!RUNS && e >= a.V) break;  // (uniform)
        if constexpr (RUNS) s0 = s1 = 0;
        if (e >= 0 && e + SUB <= a.V) {
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const float x0 = x[i][k], x1 = x[i][k + 1];
                top = max3_abs(top, x0, x1);
                s0 = add_exp(s0, x0, c, tab);
                s1 = add_exp(s1, x1, c, tab);
            }
        } else if (!RUNS || e < a.V) {  // (an end of the row: what is -inf counts as 2^-1020)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float y = x[i][k];
                if (y > -INFINITY) top = fmaxf(top, __builtin_fabsf(y));
                s0 += exp2_steps(double(y) * c, tab);
            }
        }
        // Runs' sums over the wave, four together: two, then four of them side by side in the lanes, a row of 16 lanes each in the
        // order 0, 2, 1, 3 (one by one: 17.4 us for 8 rows of 16 sequences over 151936, so 15.8,
        // without any 15.2).
        if constexpr (RUNS && EACH == 1) {
            s = wave_sum(s0 + s1);
            if (lane == 0) put(0, s, 0.f);
        } else if constexpr (RUNS) {
            if (i % 2 == 0) {
                one = s0 + s1;
            } else if (i % 4 == 1) {
                two = join32(one, s0 + s1);
            } else {
                const double four = row_sum(join16(two, join32(one, s0 + s1)));
                if ((lane & 15) == 0) put(i - 3 + (lane >> 5) + (lane >> 4 & 1) * 2, four, 0.f);
                s += four;
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (eight at a time are enough in flight: more cost registers, and waves)
    }
    if constexpr (!RUNS) s = s0 + s1;
    else if (EACH > 1) s = join16(s, s), s = join32(s, s);
    // (a NaN makes the sum one; a lane past the row's end has top -1)
    const bool near = c > 0.0 && double(top) * c < FAR && s == s;
    if (__builtin_amdgcn_ballot_w64(!near) != 0 || __builtin_amdgcn_ballot_w64(top >= 0.f) == 0) {  // (uniform in the wave)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the runs above are written before they are again)
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
            if (zero) ref = 0.f;
#pragma unroll 1
            for (int i = 0; i < EACH; ++i) {
                const Piece<E> y = piece_at<E>(row, a.V, at0<EACH>(slice, i, shift), true);
                double si = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) si += exp2_steps((double(clean(y[k])) - less) * c, tab);
                if constexpr (RUNS) {
                    si = wave_sum(si);
                    if (lane == 0) put(i, si, ref);
                }
                s += si;
            }
        } else if constexpr (RUNS) {
            for (int i = lane; i < EACH; i += 64) put(i, 0.0, -INFINITY);
        }
    }
    if constexpr (!RUNS) s = wave_sum(s);
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
        const double e = exp2_steps((double(fminf(x, 3.402823466e38f)) - ref) * c, tab);
        return x >= cut && !none ? e * z : 0.0;
    }
};

// row t's token and parent (thread t): what can be reached
__device__ __forceinline__ void row_at(const VerifyArgs& a, int b, int t, int64_t& x, int& parent) {
    x = a.tokens[int64_t(b) * a.R + t];
    parent = t == 0 ? -1 : a.parent ? a.parent[int64_t(b) * a.R + t] : t - 1;
    if (!(t > 0 && x >= 0 && x < a.V && parent >= 0 && parent < t)) x = parent = -1;
}

// What a sequence's walk leaves in LDS.
struct Tree {
    double z[2 * MAX_ROWS], share[MAX_ROWS];  // 1 / the rows' sums (the draft's behind the target's)
    int64_t tok[MAX_ROWS];
    float ref[2 * MAX_ROWS];
    int best[2 * MAX_ROWS], up[MAX_ROWS], took[MAX_ROWS], line[MAX_ROWS];
    int row, n;  // the row that answers, the accepted ones with row 0 (in line)
};
// By THREADS threads, all of them; tab: filled here.
template <class E, bool DRAFT, int THREADS>
__device__ __forceinline__ void walk(const VerifyArgs& a, int b, double c, double* tab, Tree& tree) {
    const int t = threadIdx.x;
    const bool cold = greedy(a, b);
    // thread r: row r's token, its parent, and the token's logits there
    int64_t x = -1;
    int parent = -1;
    float own_p = -INFINITY, own_q = -INFINITY;
    double own_u = 0;
    if (t < a.R) {
        row_at(a, b, t, x, parent);
        tree.tok[t] = x;
        tree.up[t] = parent;
        tree.took[t] = -1;
        if (parent >= 0) {
            own_p = E::f32(row_of<E>(a, b, parent)[x]);
            if (DRAFT) own_q = E::f32(row_of<E>(a, b, a.R + parent)[x]);
            own_u = a.uniform[int64_t(b) * (a.R + 1) + parent];
        }
    }
    fill_table<THREADS>(tab);
    __syncthreads();
    // 16 lanes a row: its reference and sum out of the slices', four of them in flight
    for (int r = t >> 4; r < a.rows; r += THREADS / 16) {
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
            tree.ref[r] = all;
            tree.z[r] = all == -INFINITY ? 0.0 : 1.0 / s;
            tree.best[r] = all == -INFINITY ? -1 : at;
        }
    }
    __syncthreads();
    // probability of this thread's token in its parent's row (r >= R: the draft's)
    auto prob = [&](int r, float l) -> double { return cold ? (x == tree.best[r] ? 1.0 : 0.0) : Soft(c, tree.z[r], tree.ref[r]).of(l, tab); };
    if (parent >= 0) {
        bool again = false;  // (a token that a sibling ahead has tried)
        for (int s = 1; s < t && !DRAFT; ++s) again = again || (tree.up[s] == parent && tree.tok[s] == x);
        tree.share[t] = again ? 0.0 : prob(parent, own_p);
    }
    __syncthreads();
    if (parent >= 0) {
        bool ok;
        if (DRAFT) {
            ok = own_u * prob(a.R + parent, own_q) < tree.share[t];
        } else {  // the siblings ahead have [0, from)
            double from = 0;
            for (int s = 1; s < t; ++s) from += tree.up[s] == parent ? tree.share[s] : 0.0;
            ok = own_u < from + tree.share[t] && !(own_u < from);
        }
        if (ok) tree.took[parent] = t;  // (one child at most: their parts of [0, 1) do not meet)
    }
    __syncthreads();
    if (t == 0) {
        int n = 0, at = 0;
        tree.line[n++] = 0;
        while (tree.took[at] >= 0) tree.line[n++] = at = tree.took[at];  // (a child's row is behind its parent's)
        tree.row = at;
        tree.n = n;
    }
    __syncthreads();
}

template <class E, int EACH>
__global__ __launch_bounds__(NT) void verify_walk_kernel(VerifyArgs a) {
    __shared__ double tab[STEPS];
    __shared__ Tree tree;
    const int slice = int(blockIdx.x % unsigned(a.pieces)), b = int(blockIdx.x / unsigned(a.pieces));
    const int t = threadIdx.x;
    const double c = rate_of(a, b);
    walk<E, true, NT>(a, b, c, tab, tree);
    const int row = tree.row;
    const bool refused = row + 1 < a.R && tree.up[row + 1] == row, cold = greedy(a, b);
    const Answer w{tree.z[row], refused ? tree.z[a.R + row] : 0.0, tree.ref[row], refused ? tree.ref[a.R + row] : 0.f, row, refused};
    if (slice == 0) {
        if (t < a.R) a.path[int64_t(b) * a.R + t] = t < tree.n ? tree.line[t] : -1;
        if (t == 0) {
            a.count[b] = tree.n;
            a.answer[b] = w;
            if (cold) a.next[b] = tree.best[row];
        }
    }
    if (cold) return;  // (uniform)
    // the sums of every wave's runs of SUB logits, the next one's logits on their way
    const typename E::type *pr = row_of<E>(a, b, row), *qr = refused ? row_of<E>(a, b, a.R + row) : pr;
    const int shift = shift_of<E>(pr);
    const bool alike = shift == shift_of<E>(qr);  // (to the 16-byte boundaries)
    const Soft p(c, w.zp, w.rp), q(c, w.zq, w.rq);
    double* sums = a.sums + (int64_t(b) * a.pieces + slice) * (EACH * (NT / 64)) + (t >> 6);
    Piece<E> x = piece_at<E>(pr, a.V, at0<EACH>(slice, 0, shift), true), y = piece_at<E>(qr, a.V, at0<EACH>(slice, 0, shift), alike);
#pragma unroll 1
    for (int i = 0; i < EACH; ++i) {
        const Piece<E> x0 = x, y0 = y;
        if (i + 1 < EACH) {
            const int e = at0<EACH>(slice, i + 1, shift);
            x = piece_at<E>(pr, a.V, e, true);
            y = piece_at<E>(qr, a.V, e, alike);
        }
        double s = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            double v = p.of(x0[k], tab);
            if (refused) v = __builtin_fmax(v - q.of(y0[k], tab), 0.0);  // (uniform)
            s += v;
        }
        s = wave_sum(s);
        if ((t & 63) == 0) sums[i * (NT / 64)] = s;
    }
}

// ---- the draw -----------------------------------------------------------------------------------------------------
// One work-group per sequence goes through this code once: besides the loads that wait for each other its instructions' own way
// from memory counts, so there are few of them (a logit per thread and one loop for the run and the token, 5 KB, against eight logits per lane of
// one wave, 18 KB: 9.8 -> 4.9 us).
constexpr int DT = 512;  // threads of the draw: all runs of a vocabulary of 262144 at once, all logits of a run
static_assert(DT == SUB, "");
struct Scan {
    double tmp[DT / 64], aim;
    int first[DT / 64], last[DT / 64];
};
// inclusive sum over the work-group's threads in order, and the total (every thread calls it)
__device__ __forceinline__ double block_scan(double v, double& total, Scan& sc) {
    const int w = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();  // (tmp may be in use by the call before)
    if ((threadIdx.x & 63) == 63) sc.tmp[w] = v;
    __syncthreads();
    double before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < DT / 64; ++i) {
        before = i == w ? total : before;
        total += sc.tmp[i];
    }
    return v + before;
}
// The first thread whose weight, with those ahead (upto), passes `to`; `passed`: there is one; else the last that has any (-1:
// none).
__device__ __forceinline__ int pick(double v, double upto, double to, bool& passed, Scan& sc) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t any = __builtin_amdgcn_ballot_w64(v > 0), past = __builtin_amdgcn_ballot_w64(v > 0 && upto > to);
    if ((threadIdx.x & 63) == 0) {
        sc.first[w] = past ? w * 64 + __builtin_ctzll(past) : 0x7FFFFFFF;
        sc.last[w] = any ? w * 64 + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    int first = 0x7FFFFFFF, last = -1;
#pragma unroll
    for (int i = 0; i < DT / 64; ++i) {
        first = min(first, sc.first[i]);
        last = max(last, sc.last[i]);
    }
    passed = first < DT;
    return passed ? first : last;
}
// The same over more runs than threads: sum_at(i), 0 behind the last. The aim within the run goes to sc.aim.
template <class F>
__device__ int pick_long(F sum_at, int runs, double u, Scan& sc) {
    const int t = threadIdx.x;
    double total = 0, before = 0, part;
    for (int i0 = 0; i0 < runs; i0 += DT) {
        block_scan(sum_at(i0 + t), part, sc);
        total += part;
    }
    const double to = u * total;
    int found = -1;
    for (int i0 = 0; i0 < runs; i0 += DT) {
        const double s = sum_at(i0 + t), upto = before + block_scan(s, part, sc);
        before += part;
        bool passed;
        const int at = pick(s, upto, to, passed, sc);
        if (at == t) sc.aim = to - (upto - s);  // (of the last with any as long as none passes)
        if (at >= 0) found = i0 + at;
        if (passed) break;  // (uniform)
    }
    __syncthreads();
    return found;
}
// The weight of a logit of the row that answers.
template <class E>
struct Weight {
    const typename E::type *p, *q;
    Soft sp, sq;
    int V;
    bool rest;
    __device__ __forceinline__ Weight(const VerifyArgs& a, int b, const Answer& w, double c)
        : p(row_of<E>(a, b, w.row)), q(w.refused ? row_of<E>(a, b, a.R + w.row) : p), sp(c, w.zp, w.rp), sq(c, w.zq, w.rq), V(a.V), rest(w.refused) {}
    struct Logit {
        typename E::type x, y;
        bool in;
    };
    __device__ __forceinline__ Logit load(int e) const {
        const bool in = e >= 0 && e < V;
        return {p[in ? e : 0], q[in ? e : 0], in};
    }
    __device__ __forceinline__ double of(const Logit& l, const double* tab) const {
        double v = sp.of(E::f32(l.x), tab);
        if (rest) v = __builtin_fmax(v - sq.of(E::f32(l.y), tab), 0.0);  // (uniform)
        return l.in ? v : 0.0;
    }
    __device__ __forceinline__ double at(int e, const double* tab) const { return of(load(e), tab); }
};
// The draw: of the runs, then of the run's logits. mine: sum_at(t); weight(e): logit e's; none(): nothing has any, true: sum_at has
// changed.
template <class F, class G, class N>
__device__ __forceinline__ int64_t drawn(double mine, F sum_at, int runs, double u, int shift, G weight, N none, Scan& sc) {
    const int t = threadIdx.x;
    int e0 = 0;  // level 1: the run's first logit
    bool runs_left = true;
#pragma unroll 1
    for (double v = mine;;) {
        int at;
        if (runs_left && runs > DT) {
            at = pick_long(sum_at, runs, u, sc);
        } else {
            double total;
            const double upto = block_scan(v, total, sc), to = runs_left ? u * total : sc.aim;
            bool passed;
            at = pick(v, upto, to, passed, sc);
            if (runs_left && at == t) sc.aim = to - (upto - v);
        }
        if (!runs_left) return at < 0 ? -1 : e0 + at;  // (a run with a sum has a logit with a weight)
        if (at < 0) {
            if (!none()) return -1;
            v = sum_at(t);
            continue;
        }
        runs_left = false;
        e0 = at * SUB - shift;
        v = weight(e0 + t);
    }
}

template <class E>
__global__ __launch_bounds__(DT) void verify_draw_kernel(VerifyArgs a, int runs) {
    __shared__ double tab[STEPS];
    __shared__ Scan sc;
    const int t = threadIdx.x, b = int(blockIdx.x);
    const double c = rate_of(a, b);
    if (greedy(a, b)) return;  // (uniform: the walk has written the answer)
    double* sums = a.sums + int64_t(b) * runs;
    auto sum_at = [&](int i) { return i < runs ? sums[i] : 0.0; };
    const double mine = sum_at(t);
    const Answer w = a.answer[b];
    const double u = a.uniform[int64_t(b) * (a.R + 1) + a.R];
    fill_table<DT>(tab);
    Weight<E> weight(a, b, w, c);
    const int shift = shift_of<E>(weight.p);
    const int64_t x = drawn(mine, sum_at, runs, u, shift, [&](int e) { return weight.at(e, tab); }, [&]() {
        if (!weight.rest) return false;
        weight.rest = false;  // nothing is left of p - q: the answer is p's
#pragma unroll 1
        for (int i = t >> 6; i < runs; i += DT / 64) {
            double s = 0;
#pragma unroll 1
            for (int j = t & 63; j < SUB; j += 64) s += weight.at(i * SUB - shift + j, tab);
            s = wave_sum(s);
            if ((t & 63) == 0) sums[i] = s;
        }
        __syncthreads();
        return true;
    }, sc);
    if (t == 0) a.next[b] = x;
}

// Without drafts' probabilities: the walk and the draw. The runs' sums are the rows kernel's, but those with a child's token,
// which are taken again without it (subtracted, a likely child would leave its rounding).
constexpr double LEAST_RUN = 0x1p-1009;  // a run's sum that counts as none: all its logits could be ones that do
template <class E>
__global__ __launch_bounds__(DT) void verify_answer_kernel(VerifyArgs a, int per_row) {
    __shared__ double tab[STEPS], less[MAX_ROWS], part[MAX_ROWS][DT / 64];
    __shared__ int child[MAX_ROWS], children;
    __shared__ Tree tree;
    __shared__ Scan sc;
    const int t = threadIdx.x, b = int(blockIdx.x);
    const double c = rate_of(a, b);
    const double u = a.uniform[int64_t(b) * (a.R + 1) + a.R];
    walk<E, false, DT>(a, b, c, tab, tree);
    const int row = tree.row;
    if (t < a.R) a.path[int64_t(b) * a.R + t] = t < tree.n ? tree.line[t] : -1;
    if (t == 0) a.count[b] = tree.n;
    if (greedy(a, b)) {  // (uniform)
        if (t == 0) a.next[b] = tree.best[row];
        return;
    }
    const Weight<E> weight(a, b, Answer{tree.z[row], 0.0, tree.ref[row], 0.f, row, 0}, c);
    const int shift = shift_of<E>(weight.p), runs = (a.V + shift + SUB - 1) / SUB;
    const Part* run = a.run + (int64_t(b) * a.R + row) * per_row;
    Part first{0.0, -INFINITY, 0};  // (on its way while the children's runs are)
    if (t < runs) first = run[t];
    // ---- the children that were tried, and the sums of their runs without them
    if (t < 64) {
        const bool is = t < a.R && tree.up[t] == row;
        const uint64_t m = __builtin_amdgcn_ballot_w64(is);
        if (is) child[__popcll(m & ((uint64_t(1) << t) - 1))] = int(tree.tok[t]);
        if (t == 0) children = __popcll(m);
    }
    __syncthreads();
    const int kids = children;
    auto without = [&](int e, double v) {
#pragma unroll 1
        for (int k = 0; k < kids; ++k) v = child[k] == e ? 0.0 : v;
        return v;
    };
    if (kids > 0) {  // (uniform)
        auto at = [&](int k) { return (child[k] + shift) / SUB * SUB - shift + t; };  // this thread's logit of child k's run
        auto next = weight.load(at(0));
#pragma unroll 1
        for (int k = 0; k < kids; ++k) {
            const auto l = next;
            next = weight.load(at(min(k + 1, kids - 1)));
            const double s = wave_sum(without(at(k), weight.of(l, tab)));
            if ((t & 63) == 0) part[k][t >> 6] = s;
        }
        __syncthreads();
        if (t < kids) {
            double s = 0;
#pragma unroll
            for (int w = 0; w < DT / 64; ++w) s += part[t][w];
            less[t] = s;
        }
        __syncthreads();
    }
    // (Of a run whose reference is 2^1020 or more below the row's nothing is left, 2^-111 at most; the exponential, which ends at
    // 2^-1020, would leave a sum where no logit has a weight.)
    auto sum_of = [&](int i, const Part& p) {
        const double down = (double(p.ref) - weight.sp.ref) * c;
        double s = p.ref == weight.sp.ref ? p.sum : !(down > LEAST) ? 0.0 : p.sum * exp2_steps(down, tab);
        s = s >= LEAST_RUN ? s * weight.sp.z : 0.0;
#pragma unroll 1
        for (int k = 0; k < kids; ++k) s = (child[k] + shift) / SUB == i ? less[k] : s;
        return s;
    };
    const int64_t x = drawn(t < runs ? sum_of(t, first) : 0.0, [&](int i) { return i < runs ? sum_of(i, run[i]) : 0.0; }, runs, u, shift,
                            [&](int e) { return without(e, weight.at(e, tab)); }, [&]() { return false; }, sc);
    if (t == 0) a.next[b] = x;
}

template <class E, int ROWS, int WALK>
int launch(const VerifyArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((verify_rows_kernel<E, ROWS, false>), dim3(unsigned(int64_t(a.slices) * a.rows * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_walk_kernel<E, WALK>), dim3(unsigned(a.pieces * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_draw_kernel<E>), dim3(unsigned(a.B)), dim3(DT), 0, st, a, a.pieces * WALK * (NT / 64));
    MDX_LAUNCHED();
    return MDX_OK;
}
template <class E, int ROWS>
int launch_rows(const VerifyArgs& a, int walk, hipStream_t st) {
    if (a.draft) return walk == 4 ? launch<E, ROWS, 4>(a, st) : walk == 2 ? launch<E, ROWS, 2>(a, st) : launch<E, ROWS, 1>(a, st);
    hipLaunchKernelGGL((verify_rows_kernel<E, ROWS, true>), dim3(unsigned(int64_t(a.slices) * a.rows * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_answer_kernel<E>), dim3(unsigned(a.B)), dim3(DT), 0, st, a, a.slices * ROWS * (NT / 64));
    MDX_LAUNCHED();
    return MDX_OK;
}
template <class E>
int launch_any(const VerifyArgs& a, int rows, int walk, hipStream_t st) {
    return rows == 8 ? launch_rows<E, 8>(a, walk, st) : rows == 4 ? launch_rows<E, 4>(a, walk, st) : launch_rows<E, 1>(a, walk, st);
}

int64_t slices_of(int64_t V, int each) { return (V + 7 + slice_of(each) - 1) / slice_of(each); }
// Pieces of eight logits per thread: as many as leave work-groups enough (their exponentials are a chain of 2 us).
int rows_each(int64_t B, int64_t rows, int64_t V) { return B * rows * slices_of(V, 8) >= 2048 ? 8 : B * rows * slices_of(V, 4) >= 1024 ? 4 : 1; }
// (the walk, over 151936: 32 sequences 17.2 us with one, 16.0 with two, 17.4 with four; 64: 24.0 with two, 21.9 with four)
int walk_each(int64_t B, int64_t V) { return B * slices_of(V, 1) > 4096 ? 4 : B * slices_of(V, 1) > 2048 ? 2 : 1; }
bool fits(int64_t B, int64_t rows, int64_t V) { return B * rows * slices_of(V, rows_each(B, rows, V)) <= most_groups(NT); }  // (of a walk's pieces there are fewer)
int64_t runs_of(int64_t V, int each) { return slices_of(V, each) * each * (NT / 64); }  // (a multiple of 4)

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_verify_drafts_workspace(int64_t B, int64_t R, int64_t V, int32_t drafted) {
    if (B < 1 || B > 1024 || R < 1 || R > MAX_ROWS || V < 1 || V >= (int64_t(1) << 24)) return 0;
    const int64_t rows = drafted ? 2 * R - 1 : R;
    if (!fits(B, rows, V)) return 0;
    const int each = rows_each(B, rows, V);
    const size_t parts = size_t(B * rows * slices_of(V, each)) * sizeof(Part);
    return parts + (drafted ? size_t(B * runs_of(V, walk_each(B, V))) * 8 + size_t(B) * sizeof(Answer) : size_t(B * R * runs_of(V, each)) * sizeof(Part));
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
    MDX_CHECK(fits(B, drafted ? 2 * R - 1 : R, V), "too many rows times logits for one call");
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
    a.part = static_cast<Part*>(workspace);
    if (drafted) {
        a.sums = reinterpret_cast<double*>(a.part + B * a.rows * a.slices);
        a.answer = reinterpret_cast<Answer*>(a.sums + B * runs_of(V, walk));
    } else {
        a.run = a.part + B * a.rows * a.slices;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MDX_DT_BF16) return launch_any<Bf>(a, rows, walk, st);
    if (dtype == MDX_DT_F16) return launch_any<Hf>(a, rows, walk, st);
    return launch_any<Ff>(a, rows, walk, st);
}
