// What the paged cache's bookkeeping shares: the free pages, a page's mean key (layout: mdx_pages.hip).
#pragma once
#include "mdx_common.hpp"

namespace mdx {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int PLAN_T = 1024;      // threads of the planning work-group
constexpr int MAX_SEQS = 1024;    // pairs of a fork or an eviction, sequences of a commit: one planning thread each

// ---- the free pages -------------------------------------------------------------------------------------
// Inclusive sum over a wave's lanes in order, by DPP: the lane 1, 2, 4, 8 ahead in its row of 16, then the rows' last lanes (the
// LDS crossbar's steps are six times as long).
template <int CTRL, int ROWS>
__device__ __forceinline__ int lane_ahead(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_sum_incl(int v) {
    v += lane_ahead<0x111, 0xF>(v);
    v += lane_ahead<0x112, 0xF>(v);
    v += lane_ahead<0x114, 0xF>(v);
    v += lane_ahead<0x118, 0xF>(v);
    v += lane_ahead<0x142, 0xA>(v);
    v += lane_ahead<0x143, 0xC>(v);
    return v;
}

// Inclusive sum over the work-group's threads (16 waves), and the total; `tmp` of 16 ints. Every thread calls it.
__device__ __forceinline__ int block_sum_incl(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = wave_sum_incl(v);
    __syncthreads();  // (tmp may be in use by the call before)
    if (lane == 63) tmp[w] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < PLAN_T / 64; ++i) {
        const int x = tmp[i];
        before += i < w ? x : 0;
        total += x;
    }
    return v + before;
}

// The lowest free pages into list, `want` of them at most, in order; how many there are. Threads take 16 neighbouring
// references each (one round of loads in flight per 16384 pages) and stop at the round that has enough.
__device__ int free_pages(const int32_t* refs, int P, int want, int32_t* list, int* tmp) {
    constexpr int PER = 16;
    int found = 0;
    for (int p0 = 0; p0 < P && found < want; p0 += PLAN_T * PER) {  // (uniform)
        const int at = p0 + int(threadIdx.x) * PER;
        int r[PER];
        if (at + PER <= P && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) *reinterpret_cast<int4*>(r + i) = *reinterpret_cast<const int4*>(refs + at + i);
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) r[i] = at + i < P ? refs[at + i] : 1;
        }
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) n += r[i] == 0;
        int total;
        int to = found + block_sum_incl(n, tmp, total) - n;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (r[i] == 0) {
                if (to < want) list[to] = at + i;
                ++to;
            }
        found += total;
    }
    return found < want ? found : want;
}

__device__ __forceinline__ int clamp_len(int n, int W, int lt) {
    const int most = W << lt;
    return n < 0 ? 0 : (n > most ? most : n);
}

__device__ __forceinline__ float el(uint16_t x, int half) { return half ? fp16_to_f32(x) : bf2f(x); }
__device__ __forceinline__ uint16_t to_el(float f, int half) {
    return half ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)) : f2bf(f);
}

// The mean of T rows of D elements at `keys` (the cache or LDS), to `mean`, by one wave: a lane holds eight dims of every
// (64 / (D / 8))-th row, fp32 sums, the row groups joined by lane exchanges, one rounding to the cache's type.
__device__ __forceinline__ void mean_rows(const uint16_t* keys, uint16_t* mean, int T, int D, int half, int lane) {
    const int lanes = D / 8, step = 64 / lanes, sub = lane / lanes, d8 = lane % lanes * 8;
    const float inv = 1.f / float(T);  // (a power of two: exact)
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
#pragma unroll 8
    for (int r = sub; r < T; r += step) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(keys + int64_t(r) * D + d8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[2 * i] += el(uint16_t(v[i] & 0xFFFFu), half);
            s[2 * i + 1] += el(uint16_t(v[i] >> 16), half);
        }
    }
    for (int d = lanes; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += __shfl_xor(s[i], d, 64);
    if (sub == 0) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = unsigned(to_el(s[2 * i] * inv, half)) | (unsigned(to_el(s[2 * i + 1] * inv, half)) << 16);
        *reinterpret_cast<u32x4*>(mean + d8) = o;
    }
}
// The mean key of page e in chunk kc (layer, kv head), by one wave.
template <class Args>
__device__ void mean_key(const Args& a, int64_t kc, int e, int lane) {
    const int64_t layer = kc / a.Hk, h = kc % a.Hk;
    mean_rows(reinterpret_cast<const uint16_t*>(a.kv) + (((layer * 2 * a.Hk + h) * a.P + e) << a.lt) * a.D, a.ksum + (kc * a.P + e) * a.D, a.T, a.D, a.half,
              lane);
}

int log2_of(int64_t T) {
    for (int i = 4; i <= 10; ++i)
        if (T == int64_t(1) << i) return i;
    return -1;
}

}  // namespace
}  // namespace mdx
