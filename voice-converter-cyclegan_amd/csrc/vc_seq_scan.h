// vc_seq_scan.h -- the selective state space scan: how lanes, tiles and utterances are laid out, shared by its forward and backward kernels.
//
//   h[t][n] = exp(delta[t] A[n]) h[t-1][n] + delta[t] x[t] B[t][n];   y[t] = sum_n C[t][n] h[t][n] + D x[t], gated by z sigmoid(z)
//
// Lanes.  L lanes share one channel, each holds NS of its states in registers (L * NS = NP >= states), so a wave holds 64 / L channels and a
// sum over the states is NS additions and a few lane exchanges.  What depends on the channel alone (softplus, its slope, the gate) would be
// worked out L times over: instead rows go in batches of L, lane j of a channel works out row j of the batch, and the recurrence fetches row i's
// value from lane i.  B and C of a tile lie in LDS as fp32, one private copy for each wave, so the waves of a block need no barrier for them.
//
// Tiles.  TILE rows of one utterance (the last tile of an utterance may be short; rows it lacks get delta = 0, which leaves the state as it is).
// Tiles are numbered by slots: utterance s owns the slots from begin(s) / TILE + s on, which needs no sum over the lengths of those before it
// and never overlaps; a few slots stay empty.
#pragma once
#include "vc_seq.h"

constexpr int TILE = 16;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct ScanK {
    vc_scan_args a; SeqMap m;
    int cg, nblk;                  // channels of a group; blocks that cover them
    int slots;                     // slots in all
    float *part, *dapart, *chpart; // backward: partial sums of dB / dC, dA, and of dD and ddt_bias
};

__device__ __forceinline__ int slot_base(const SeqMap& m, int s) { return seq_begin(m, s) / TILE + s; }

template <int I, int N, class F> __device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) { f(std::integral_constant<int, I>()); static_for<I + 1, N>(f); }
}
// lane i's value of the L lanes that share a channel
template <int L, int I> __device__ __forceinline__ float from_lane(float v) {
    if constexpr (L == 4) return dpp_read<I * 0x55>(v);          // quad_perm [i,i,i,i]
    else return dpp_read<0x150 + I>(v);                          // row_newbcast:i
}
// one step of sums_by_row: rows kept by bit BIT of the lane, the others handed to the lane that keeps them
template <int CTRL, int N> __device__ __forceinline__ void halve(float (&v)[N], bool up) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float keep = up ? v[i + N / 2] : v[i], send = up ? v[i] : v[i + N / 2];
        v[i] = keep + dpp_read<CTRL>(send);
    }
}
// v[i] = this lane's share of row i; lane j gets the sum of row j over the L lanes (L - 1 additions in place of L log2 L)
template <int L> __device__ __forceinline__ float sums_by_row(float (&v)[L], int j) {
    if constexpr (L == 16) {
        halve<0x128, 16>(v, j & 8);                              // row_ror:8
        float w[8], q[4], p[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = v[i];
        halve<0x141, 8>(w, j & 4);                               // row_half_mirror
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = w[i];
        halve<0x4E, 4>(q, j & 2);
        p[0] = q[0]; p[1] = q[1];
        halve<0xB1, 2>(p, j & 1);
        return p[0];
    } else {
        float p[2];
        halve<0x4E, 4>(v, j & 2);                                // quad_perm [2,3,0,1]
        p[0] = v[0]; p[1] = v[1];
        halve<0xB1, 2>(p, j & 1);                                // quad_perm [1,0,3,2]
        return p[0];
    }
}
// sum over the L lanes of a channel, in all of them
template <int L> __device__ __forceinline__ float channel_sum(float v) {
    if constexpr (L == 16) return row16_sum(v);
    v += dpp_read<0xB1>(v);
    return v + dpp_read<0x4E>(v);
}

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) in (0, 1], and its slope.  log(1 + e) = 2 atanh(e / (2 + e)) by its series: the argument is at
// most 1/3, seven terms leave 1.4e-8, and a small e keeps all its bits (a logarithm of the rounded 1 + e would lose them: steps of 0.001 are ordinary here)
__device__ __forceinline__ float softplus(float v, float& slope) {
    const float e = expf(-fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 1.f / 13.f;
    p = fmaf(p, q, 1.f / 11.f); p = fmaf(p, q, 1.f / 9.f); p = fmaf(p, q, 1.f / 7.f); p = fmaf(p, q, 1.f / 5.f); p = fmaf(p, q, 1.f / 3.f); p = fmaf(p, q, 1.f);
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    slope = v >= 0.f ? r : e * r;
    return fmaxf(v, 0.f) + 2.f * s * p + (v - v);                // v - v: a NaN stays one (fmaxf drops it)
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Rows [row0, row0 + nr) of B or C (group g) as fp32 into dst[TILE][NP]: four lanes a row, NP / 4 states each; zeros where there is no row or state
template <class T, int NP> __device__ __forceinline__ void stage_states(const T* src, int64_t ld, int row0, int nr, int states, float* dst, int lane) {
    constexpr int W = NP / 4;
    const int r = lane >> 2, n = (lane & 3) * W;
    float f[W];
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = 0.f;
    if (r < nr) load_some<T, W>(src + (int64_t)(row0 + r) * ld + n, f, states - n);
#pragma unroll
    for (int i = 0; i < W; ++i) dst[r * NP + n + i] = f[i];
}
// LDS of one wave: what its lanes wrote is there for all of them (the hardware keeps a wave's LDS accesses in order; this keeps the compiler's)
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Where a lane works
template <int L, int NS> struct Lane {
    int lane, wave, j, c, n0, nn; bool ok; int g;
    __device__ __forceinline__ Lane(const ScanK& k, int waves, int blk) {
        lane = threadIdx.x & 63; wave = threadIdx.x >> 6;
        j = lane % L;
        g = blk / k.nblk;
        const int cw = 64 / L, cb = (blk - g * k.nblk) * waves * cw + wave * cw + lane / L;
        ok = cb < k.cg;
        c = g * k.cg + min(cb, k.cg - 1);
        n0 = j * NS;
        nn = max(0, min(NS, k.a.states - n0));
    }
};
template <int NS> __device__ __forceinline__ void load_state(const float* p, float (&h)[NS], int nn) { load_some<float, NS>(p, h, nn); }

// which register layout serves a number of states, and how many channels a block of `waves` waves covers
#define SCAN_LAYOUT(T, states, F, ...) \
    ((states) <= 8 ? F<T, 4, 2>(__VA_ARGS__) : (states) <= 16 ? F<T, 4, 4>(__VA_ARGS__) : (states) <= 32 ? F<T, 16, 2>(__VA_ARGS__) : F<T, 16, 4>(__VA_ARGS__))
static inline int scan_lanes(int states) { return states <= 16 ? 4 : 16; }
static inline int scan_padded(int states) { return states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }
int scan_setup(const char* who, const vc_scan_args* a, bool bwd, ScanK* k);
