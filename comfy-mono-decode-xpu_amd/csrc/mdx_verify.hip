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
// Two launches. verify_rows_kernel: a work-group per 8192 logits of a row takes their maximum M and sum of exp((x - M) / T).
// verify_draw_kernel: a work-group per 8192 logits of a sequence joins the rows' parts, walks the tree (every work-group of a
// sequence alike, from LDS), takes the weights of its piece of the row that answers; the last one done finds the piece that
// the draw falls in and the token in it.
//
// What bounds it: the logits' bytes, each read once (the row that answers again, out of the caches), and at about the same rate
// the exponentials (18 vector instructions each, float64 at the rate of float32 on this chip).
// Exponentials: 2^(a / 32) = table[k % 32] 2^(k / 32) poly(a - k), k = rint(a); a table of 32 doubles is one LDS line of banks, so
// no two different entries meet in one; the polynomial of degree 4 interpolates at the Chebyshev points of [-1/2, 1/2]
// (8e-14 relative).
//
// Reference: the walk's role is csrc/mtp_loop.sycl:86-196's accept (which compares with one sampled token per row).
#include "mdx_common.hpp"

namespace mdx {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_ROWS = 64;
constexpr int NT = 256;
constexpr int EACH = 4;               // pieces of 8 logits per thread
constexpr int SLICE = NT * EACH * 8;  // logits of a work-group

struct Part {  // of a slice of a row
    double sum;   // sum of exp((x - top) / T)
    float top;    // -inf: nothing there
    int32_t at;   // the lowest index of top (T = 0 alone)
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
    double* sums;    // [B][slices]
    int32_t* done;   // [B]
    int B, R, V, slices, rows;  // rows: of a sequence, the draft's behind the target's
};

// ---- exponentials -----------------------------------------------------------------------------------------
__device__ __forceinline__ void fill_table(double* tab) {  // (the caller's barrier follows)
    if (threadIdx.x < 32) tab[threadIdx.x] = exp2(double(threadIdx.x) / 32.0);
}
// 2^(a / 32); below 2^-1021 (NaN too) that
__device__ __forceinline__ double exp2_32(double a, const double* tab) {
    a = __builtin_fmax(a, -32.0 * 1021.0);
    const double t = a + 6755399441055744.0;  // 1.5 2^52: the low word is rint(a)
    const int k = __double2loint(t);
    const double f = a - (t - 6755399441055744.0);
    double p = __builtin_fma(f, 0x1.3b2b1bee88b09p-27, 0x1.c6b167e571135p-20);
    p = __builtin_fma(p, f, 0x1.ebfbdff8131c3p-13);
    p = __builtin_fma(p, f, 0x1.62e42fef6d01ap-6);
    p = __builtin_fma(p, f, 1.0);
    const double v = tab[k & 31];
    return p * __hiloint2double(__double2hiint(v) + ((k & ~31) << 15), __double2loint(v));
}
// 32 log2(e) / T, 0 for the largest logit alone (T of infinity: nearly 0, all logits alike but those of -inf)
__device__ __forceinline__ double rate_of(const VerifyArgs& a, int b) {
    const float t = a.heat ? a.heat[b] : a.one_heat;
    return t > 0.f ? __builtin_fmax(32.0 * 1.4426950408889634074 / double(t), 1e-300) : 0.0;
}
__device__ __forceinline__ bool greedy(const VerifyArgs& a, int b) { return !((a.heat ? a.heat[b] : a.one_heat) > 0.f); }

// ---- logits -----------------------------------------------------------------------------------------------
struct Bf {
    typedef uint16_t type;
    static __device__ __forceinline__ float f32(uint16_t x) { return bf2f(x); }
};
struct Hf {
    typedef uint16_t type;
    static __device__ __forceinline__ float f32(uint16_t x) { return fp16_to_f32(x); }
};
struct Ff {
    typedef float type;
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

// This thread's pieces of slice `slice`: x[i][k] is logit at0(i) + k, -inf outside of the row.
template <class E>
__device__ __forceinline__ int at0(int slice, int i, int shift) {
    return (slice * (NT * EACH) + i * NT + int(threadIdx.x)) * 8 - shift;
}
template <class E>
__device__ __forceinline__ void load(const typename E::type* row, int V, int slice, float (&x)[EACH][8]) {
    typedef typename E::type T;
    const int shift = shift_of<E>(row);
    constexpr int W = sizeof(T) * 8 / 16;  // 16-byte words of a piece
    u32x4 v[EACH][W];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = at0<E>(slice, i, shift);
        if (e >= 0 && e + 8 <= V) {
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = *reinterpret_cast<const u32x4*>(row + e + j * (16 / int(sizeof(T))));
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = at0<E>(slice, i, shift);
        if (e >= 0 && e + 8 <= V) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (sizeof(T) == 2) x[i][k] = E::f32(uint16_t(v[i][0][k / 2] >> (16 * (k & 1))));
                else x[i][k] = __uint_as_float(v[i][k / 4][k & 3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[i][k] = e + k >= 0 && e + k < V ? E::f32(row[e + k]) : -INFINITY;
        }
    }
}

// ---- the rows' maxima and sums --------------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

template <class E>
__global__ __launch_bounds__(NT) void verify_rows_kernel(VerifyArgs a) {
    __shared__ double tab[32], sum_w[NT / 64];
    __shared__ float top_w[NT / 64];
    __shared__ int at_w[NT / 64];
    const int slice = int(blockIdx.x % unsigned(a.slices)), r = int(blockIdx.x / unsigned(a.slices)) % a.rows,
              b = int(blockIdx.x / unsigned(a.slices)) / a.rows;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const typename E::type* row = row_of<E>(a, b, r);
    float x[EACH][8];
    load<E>(row, a.V, slice, x);
    fill_table(tab);
    if (slice == 0 && r == 0 && threadIdx.x == 0) a.done[b] = 0;
    const double c = rate_of(a, b);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, x[i][k]);
    top = wave_max(top);
    if (top == INFINITY) {  // (uniform in the wave)
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) x[i][k] = clean(x[i][k]);
        top = clean(top);
    }
    __syncthreads();  // (the table)
    double s0 = 0, s1 = 0;
    int at = 0x7FFFFFFF;
    if (c == 0.0) {
        const int shift = shift_of<E>(row);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (x[i][k] == top && top > -INFINITY) at = min(at, at0<E>(slice, i, shift) + k);
        for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d, 64));
    } else if (top > -INFINITY) {  // (uniform in the wave)
        const double m = double(top);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                s0 += exp2_32((double(x[i][k]) - m) * c, tab);
                s1 += exp2_32((double(x[i][k + 1]) - m) * c, tab);
            }
    }
    const double s = wave_sum(s0 + s1);
    if (lane == 0) {
        sum_w[w] = s;
        top_w[w] = top;
        at_w[w] = at;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    float all = top_w[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) all = fmaxf(all, top_w[i]);
    double sum = 0;
    int first = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        if (top_w[i] == -INFINITY) continue;
        sum += sum_w[i] * exp2_32((double(top_w[i]) - double(all)) * c, tab);
        if (top_w[i] == all) first = min(first, at_w[i]);
    }
    a.part[(int64_t(b) * a.rows + r) * a.slices + slice] = Part{sum, all, first};
}

// ---- the walk and the draw ------------------------------------------------------------------------------------
// Inclusive sum over the work-group's threads in order, and the total; `tmp` of NT / 64 doubles. Every thread calls it.
__device__ __forceinline__ double block_scan(double v, double* tmp, double& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double u = __shfl_up(v, d, 64);
        if (lane >= d) v += u;
    }
    __syncthreads();  // (tmp may be in use by the call before)
    if (lane == 63) tmp[w] = v;
    __syncthreads();
    double before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        if (i < w) before += tmp[i];
        total += tmp[i];
    }
    return v + before;
}

template <class E>
__global__ __launch_bounds__(NT) void verify_draw_kernel(VerifyArgs a) {
    __shared__ double tab[32], z[2 * MAX_ROWS], share[MAX_ROWS], tmp[NT / 64];
    __shared__ float top[2 * MAX_ROWS];
    __shared__ int best[2 * MAX_ROWS], up[MAX_ROWS], took[MAX_ROWS], line[MAX_ROWS], pick[2], arrived;
    __shared__ int64_t tok[MAX_ROWS];
    __shared__ double aim;
    const int slice = int(blockIdx.x % unsigned(a.slices)), b = int(blockIdx.x / unsigned(a.slices));
    const int t = threadIdx.x;
    const double c = rate_of(a, b);
    const bool cold = greedy(a, b);
    fill_table(tab);
    // thread r: row r's token, its parent, and the token's logits there
    float own_p = -INFINITY, own_q = -INFINITY;
    if (t < a.R) {
        const int64_t x = a.tokens[int64_t(b) * a.R + t];
        const int parent = t == 0 ? -1 : a.parent ? a.parent[int64_t(b) * a.R + t] : t - 1;
        const bool live = t > 0 && x >= 0 && x < a.V && parent >= 0 && parent < t;
        tok[t] = live ? x : -1;
        up[t] = live ? parent : -1;
        took[t] = -1;
        if (live) {
            own_p = clean(E::f32(row_of<E>(a, b, parent)[x]));
            if (a.draft) own_q = clean(E::f32(row_of<E>(a, b, a.R + parent)[x]));
        }
    }
    __syncthreads();
    // 16 lanes a row: its maximum and sum out of the slices'
    for (int r = t >> 4; r < a.rows; r += NT / 16) {
        const Part* part = a.part + (int64_t(b) * a.rows + r) * a.slices;
        float m = -INFINITY;
        double s = 0;
        int at = 0x7FFFFFFF;
        for (int i = t & 15; i < a.slices; i += 16) {
            const Part p = part[i];
            if (p.top == -INFINITY) continue;
            if (p.top > m) {
                s = (m == -INFINITY ? 0.0 : s * exp2_32((double(m) - double(p.top)) * c, tab)) + p.sum;
                m = p.top;
                at = p.at;
            } else {
                s += p.sum * exp2_32((double(p.top) - double(m)) * c, tab);
                if (p.top == m) at = min(at, p.at);
            }
        }
        float all = m;
        for (int d = 8; d; d >>= 1) all = fmaxf(all, __shfl_xor(all, d, 64));
        s = m == -INFINITY ? 0.0 : s * exp2_32((double(m) - double(all)) * c, tab);
        at = m == all ? at : 0x7FFFFFFF;
        for (int d = 8; d; d >>= 1) {
            s += __shfl_xor(s, d, 64);
            at = min(at, __shfl_xor(at, d, 64));
        }
        if ((t & 15) == 0) {
            top[r] = all;
            z[r] = all == -INFINITY ? 0.0 : 1.0 / s;
            best[r] = all == -INFINITY ? -1 : at;
        }
    }
    __syncthreads();
    // probability of a logit x (index v) in row r; -inf and what lies 2^1021 below the largest have none
    auto prob = [&](int r, float x, int64_t v) -> double {
        if (cold) return v == best[r] ? 1.0 : 0.0;
        const double e = (double(x) - double(top[r])) * c;
        return e >= -32.0 * 1021.0 && top[r] > -INFINITY ? exp2_32(e, tab) * z[r] : 0.0;
    };
    if (t < a.R && up[t] >= 0) {
        bool again = false;  // (a token that a sibling ahead has tried)
        for (int s = 1; s < t && !a.draft; ++s) again = again || (up[s] == up[t] && tok[s] == tok[t]);
        share[t] = again ? 0.0 : prob(up[t], own_p, tok[t]);
    }
    __syncthreads();
    if (t < a.R && up[t] >= 0) {
        const int r = up[t];
        const double u = a.uniform[int64_t(b) * (a.R + 1) + r];
        bool ok;
        if (a.draft) {
            ok = u * prob(a.R + r, own_q, tok[t]) < share[t];
        } else {  // the siblings ahead have [0, from)
            double from = 0;
            for (int s = 1; s < t; ++s) from += up[s] == r ? share[s] : 0.0;
            ok = u < from + share[t] && !(u < from);
        }
        if (ok) took[r] = t;  // (one child at most: their parts of [0, 1) do not meet)
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
    if (slice == 0) {
        if (t < a.R) a.path[int64_t(b) * a.R + t] = t < n ? line[t] : -1;
        if (t == 0) a.count[b] = n;
        if (cold && t == 0) a.next[b] = best[row];
    }
    if (cold) return;  // (uniform)

    // ---- this piece's weights of the row that answers
    const bool refused = a.draft && row + 1 < a.R && up[row + 1] == row;
    const typename E::type *pr = row_of<E>(a, b, row), *qr = refused ? row_of<E>(a, b, a.R + row) : pr;
    auto weights = [&](int sl, bool rest, double (&wt)[EACH][8]) {
        float x[EACH][8];
        load<E>(pr, a.V, sl, x);
        const int shift = shift_of<E>(pr);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) wt[i][k] = prob(row, clean(x[i][k]), 0);
        if (rest) {
            // (element by element: the two rows may stand differently to the 16-byte boundaries)
            if (shift == shift_of<E>(qr)) {
                load<E>(qr, a.V, sl, x);
            } else {
#pragma unroll
                for (int i = 0; i < EACH; ++i)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int e = at0<E>(sl, i, shift) + k;
                        x[i][k] = e >= 0 && e < a.V ? E::f32(qr[e]) : -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < EACH; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) wt[i][k] = __builtin_fmax(wt[i][k] - prob(a.R + row, clean(x[i][k]), 0), 0.0);
        } else if (!a.draft) {  // the children that were tried
            for (int s = row + 1; s < a.R; ++s) {
                if (up[s] != row) continue;
                const int e = int(tok[s]) + shift - sl * SLICE;
                if (e < 0 || e >= SLICE || (e >> 3) % NT != t) continue;
                const int i0 = (e >> 3) / NT, k0 = e & 7;
#pragma unroll
                for (int i = 0; i < EACH; ++i)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (i == i0 && k == k0) wt[i][k] = 0.0;
            }
        }
    };
    auto slice_sum = [&](const double (&wt)[EACH][8]) {
        double s = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) s += wt[i][k];
        double total;
        block_scan(s, tmp, total);
        return total;
    };
    double wt[EACH][8];
    weights(slice, refused, wt);
    const double mine = slice_sum(wt);
    if (t == 0) {
        a.sums[int64_t(b) * a.slices + slice] = mine;
        __threadfence();
        arrived = atomicAdd(a.done + b, 1);
    }
    __syncthreads();
    if (arrived != a.slices - 1) return;  // (uniform: the last one of the sequence goes on)
    __threadfence();

    // ---- the piece that the draw falls in: the sums in order, by thread 0
    const volatile double* sums = a.sums + int64_t(b) * a.slices;
    bool rest = refused;
    auto find = [&]() {
        if (t == 0) {
            double total = 0;
            for (int i = 0; i < a.slices; ++i) total += sums[i];
            aim = a.uniform[int64_t(b) * (a.R + 1) + a.R] * total;
            double before = 0, at = 0;
            int to = -1, last = -1;
            for (int i = 0; i < a.slices && to < 0; ++i) {
                const double s = sums[i];
                if (s > 0) {
                    last = i;
                    at = before;
                }
                if (before + s > aim) to = i;
                before += s;
            }
            pick[0] = to >= 0 ? to : last;
            aim -= at;
        }
        __syncthreads();
    };
    find();
    if (pick[0] < 0 && refused) {  // (uniform) nothing is left of p - q: the answer is p's
        rest = false;
        __syncthreads();
        for (int i = 0; i < a.slices; ++i) {
            weights(i, false, wt);
            const double s = slice_sum(wt);
            if (t == 0) const_cast<volatile double*>(sums)[i] = s;
        }
        __syncthreads();
        find();
    }
    const int from = pick[0];
    if (from < 0) {
        if (t == 0) a.next[b] = -1;
        return;
    }
    // ---- and the token in it
    weights(from, rest, wt);
    const int shift = shift_of<E>(pr);
    __syncthreads();
    if (t == 0) pick[0] = pick[1] = -1;
    __syncthreads();
    double before = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        double s = 0;
        int last = -1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            s += wt[i][k];
            if (wt[i][k] > 0) last = k;
        }
        double total;
        const double upto = before + block_scan(s, tmp, total), ahead = upto - s;
        if (last >= 0) {
            // the lowest whose sum passes the aim; and the last with a weight, where none does
            atomicMax(&pick[1], at0<E>(from, i, shift) + last);
            if (upto > aim) {
                double run = ahead;
                int to = -1;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    run += wt[i][k];
                    if (to < 0 && wt[i][k] > 0 && run > aim) to = k;
                }
                if (to < 0) to = last;
                const int e = at0<E>(from, i, shift) + to;
                atomicMin(reinterpret_cast<unsigned*>(&pick[0]), unsigned(e));
            }
        }
        before += total;
    }
    __syncthreads();
    if (t == 0) a.next[b] = pick[0] >= 0 ? pick[0] : pick[1];
}

template <class E>
int launch(const VerifyArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((verify_rows_kernel<E>), dim3(unsigned(int64_t(a.slices) * a.rows * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    hipLaunchKernelGGL((verify_draw_kernel<E>), dim3(unsigned(a.slices * a.B)), dim3(NT), 0, st, a);
    MDX_LAUNCHED();
    return MDX_OK;
}

int64_t slices_of(int64_t V) { return (V + 7 + SLICE - 1) / SLICE; }
size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace mdx

using namespace mdx;

extern "C" size_t mdx_verify_drafts_workspace(int64_t B, int64_t R, int64_t V, int32_t drafted) {
    if (B < 1 || B > 1024 || R < 1 || R > MAX_ROWS || V < 1 || V >= (int64_t(1) << 24)) return 0;
    const int64_t n = slices_of(V), rows = drafted ? 2 * R - 1 : R;
    return size_t(B * rows * n) * sizeof(Part) + size_t(B * n) * 8 + align16(size_t(B) * 4);
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
    a.B = int(B), a.R = int(R), a.V = int(V), a.slices = int(slices_of(V)), a.rows = int(drafted ? 2 * R - 1 : R);
    MDX_CHECK(B * a.rows * a.slices < (int64_t(1) << 30), "too many rows times logits for one call");
    a.part = static_cast<Part*>(workspace);
    a.sums = reinterpret_cast<double*>(a.part + B * a.rows * a.slices);
    a.done = reinterpret_cast<int32_t*>(a.sums + B * a.slices);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MDX_DT_BF16) return launch<Bf>(a, st);
    if (dtype == MDX_DT_F16) return launch<Hf>(a, st);
    return launch<Ff>(a, st);
}
