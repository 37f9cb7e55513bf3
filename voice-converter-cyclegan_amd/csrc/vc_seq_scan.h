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

struct ScanK {
    vc_scan_args a; SeqMap m;
    int cg, nblk, waves;           // channels of a group; blocks that cover them, and the waves of each
    int slots;                     // slots in all
    // How the time axis is shared out: items are whole utterances (chunk = 0), or runs of `chunk` slots whatever utterances these belong to.
    // In the second form a first pass works out what each run does to a state that enters it, h -> exp(A sum_delta) h + edge, and the main pass begins
    // with the sum of what the runs before it hand on.  `cut` marks the runs that hand on nothing of what enters (an utterance begins or ends there).
    int items, chunk; bool once;   // once: what enters the runs is worked out by a pass of its own
    float *edge, *sum_delta; int* cut;             // [items][cols][states], [items][cols], [items]
    float *part, *dapart, *chpart; // backward: partial sums of dB / dC, dA, and of dD and ddt_bias
};

__device__ __forceinline__ int slot_base(const SeqMap& m, int s) { return seq_begin(m, s) / TILE + s; }

// the same in all lanes, and the compiler is to know it: addresses of rows then take a scalar base
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The utterance that the slots being walked belong to
struct Cursor {
    const SeqMap& m;
    int s, base, next, begin, end, tiles;
    __device__ __forceinline__ explicit Cursor(const SeqMap& map) : m(map) {}
    __device__ __forceinline__ void load(int i) {
        s = uniform(i); begin = uniform(seq_begin(m, s)); end = uniform(seq_end(m, s, begin)); base = begin / TILE + s; tiles = (end - begin + TILE - 1) / TILE;
        next = s + 1 < m.n_seqs ? uniform(slot_base(m, s + 1)) : 0x7fffffff;
    }
    __device__ __forceinline__ void find(int q) {
        int lo = 0, hi = m.n_seqs - 1;
        while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (slot_base(m, mid) <= q) lo = mid; else hi = mid - 1; }
        load(lo);
    }
};
// the slots of an item
__device__ __forceinline__ void item_slots(const ScanK& k, int item, int& q0, int& q1) {
    if (k.chunk) { q0 = item * k.chunk; q1 = min(q0 + k.chunk, k.slots); }
    else { q0 = slot_base(k.m, item); q1 = item + 1 < k.m.n_seqs ? slot_base(k.m, item + 1) : k.slots; }
}

template <int I, int N, class F> __device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) { f(std::integral_constant<int, I>()); static_for<I + 1, N>(f); }
}
// dpp_read where every lane has a source: nothing to keep of the destination's old value, which lets the move become part of the instruction that uses it
template <int CTRL> __device__ __forceinline__ float dpp_all(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// lane i's value of the L lanes that share a channel
template <int L, int I> __device__ __forceinline__ float from_lane(float v) {
    if constexpr (L == 4) return dpp_all<I * 0x55>(v);          // quad_perm [i,i,i,i]
    else if constexpr (L == 16) return dpp_all<0x150 + I>(v);   // row_newbcast:i
    else {                                                      // row_newbcast:i, and :8 + i for the upper eight lanes of a row
        const int x = __builtin_bit_cast(int, v);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_amdgcn_mov_dpp(x, 0x150 + I, 0xf, 0xf, true), x, 0x158 + I, 0xf, 0xc, false));
    }
}
// one step of sums_by_row: rows kept by one bit of the lane, the others handed to the lane that keeps them
template <int CTRL, int N> __device__ __forceinline__ void halve(float (&v)[N], bool up) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float keep = up ? v[i + N / 2] : v[i], send = up ? v[i] : v[i + N / 2];
        v[i] = keep + dpp_all<CTRL>(send);
    }
}
// v[i] = this lane's share of row i; lane j gets the sum of row j over the L lanes (L - 1 additions in place of L log2 L)
template <int L> __device__ __forceinline__ float sums_by_row(float (&v)[L], int j) {
    if constexpr (L == 16) halve<0x128, 16>(v, j & 8);           // row_ror:8
    if constexpr (L >= 8) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = v[i];
        halve<0x141, 8>(w, j & 4);                               // row_half_mirror
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = w[i];
    }
    float q[4], p[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = v[i];
    halve<0x4E, 4>(q, j & 2);                                    // quad_perm [2,3,0,1]
    p[0] = q[0]; p[1] = q[1];
    halve<0xB1, 2>(p, j & 1);                                    // quad_perm [1,0,3,2]
    return p[0];
}
// sum over the L lanes of a channel, in all of them
template <int L> __device__ __forceinline__ float channel_sum(float v) {
    if constexpr (L == 16) return row16_sum(v);
    v += dpp_all<0xB1>(v);
    v += dpp_all<0x4E>(v);
    if constexpr (L == 8) v += dpp_all<0x141>(v);
    return v;
}

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) in [0, 1], and its slope.  log(1 + e) = 2 atanh(e / (2 + e)) by its series: the argument is at
// most 1/3, seven terms leave 1.4e-8, and a small e keeps all its bits (a logarithm of the rounded 1 + e would lose them: steps of 0.001 are ordinary here).
// dt masked by -inf or its type's lowest value is a step of exactly 0 with a slope of 0, the largest value or inf is a step of itself, a NaN stays one.
__device__ __forceinline__ float softplus(float v, float& slope) {
    const float e = exp_acc(-fminf(fabsf(v), 128.f));            // (beyond 128 it is 0 in fp32; beyond 2^127 what its argument rounds off would be no number)
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 1.f / 13.f;
    p = fmaf(p, q, 1.f / 11.f); p = fmaf(p, q, 1.f / 9.f); p = fmaf(p, q, 1.f / 7.f); p = fmaf(p, q, 1.f / 5.f); p = fmaf(p, q, 1.f / 3.f); p = fmaf(p, q, 1.f);
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    const bool below = v < 0.f;                                  // (of a NaN not: it goes on into the sum)
    slope = below ? e * r : r;
    return fmaf(2.f * s, p, below ? 0.f : v);
}

// A tensor of rows as a lane uses it: through a buffer descriptor of the tile's rows, whose bounds check gives zeros for the rows that a short tile
// lacks (where rows do not overlap) and drops stores to them, and those of lanes without a channel.  Host code keeps row strides within MAX_LD: the
// offsets in a tile fit 31 bits.
constexpr int64_t MAX_LD = 1 << 24;
template <class T, int L> struct Rows {
    const T* p; int ld, width; unsigned at, step;
    __device__ __forceinline__ Rows(const void* base, int64_t stride, int cols, int c, int j, bool ok = true)
        : p((const T*)base), ld((int)stride), width(cols * (int)sizeof(T)),
          at(ok ? (unsigned)(j * (int)stride + c) * (unsigned)sizeof(T) : 0x80000000u), step((unsigned)(L * (int)stride) * (unsigned)sizeof(T)) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(int row0, int nr) const {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)row0 * ld), 0, (nr - 1) * ld * (int)sizeof(T) + width, 0x00020000);
    }
    // rows b * L + j of a tile
    template <int NB> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t t, T (&v)[NB]) const {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (sizeof(T) == 4) v[b] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(t, at + b * step, 0, 0));
            else v[b] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(t, at + b * step, 0, 0));
        }
    }
    template <int NB> __device__ __forceinline__ void load(int row0, int nr, T (&v)[NB]) const { load(tile(row0, nr), v); }
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t t, int b, float f) const {
        if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, f), t, at + b * step, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (T)f), t, at + b * step, 0, 0);
    }
    // rows from `first` on, one after the other by the lanes of a channel
    __device__ __forceinline__ void clear(int first, int rows, int c, int j) const {
        if (at != 0x80000000u) for (int r = first + j; r < rows; r += L) ((T*)p)[(int64_t)r * ld + c] = (T)0.f;
    }
};
// A tile of B or C (a group's states contiguous): four lanes a row, NP / 4 states each, in registers until the tile before it is done with
template <class T, int NP> struct States {
    static constexpr int W = NP / 4;
    const T* p; int ld, states, r, n;
    __device__ __forceinline__ States(const void* base, int64_t stride, int g, int count, int lane) : p((const T*)base + g * count), ld((int)stride), states(count), r(lane >> 2), n((lane & 3) * W) {}
    __device__ __forceinline__ void load(int row0, int nr, T (&v)[W]) const {
        const char* base = (const char*)(p + (int64_t)row0 * ld);
        const unsigned row = (unsigned)(min(r, nr - 1) * ld) * (unsigned)sizeof(T);      // a short tile's missing rows read its last one
        if (states == NP) {
            const Pack<T, W> q = *(const Pack<T, W>*)(base + (row + n * (unsigned)sizeof(T)));
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = q.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = *(const T*)(base + (row + min(n + i, states - 1) * (unsigned)sizeof(T)));
        }
    }
    // as fp32 into dst[TILE][NP], zeros where there is no row or state
    __device__ __forceinline__ void stage(const T (&v)[W], int nr, float* dst) const {
#pragma unroll
        for (int i = 0; i < W; ++i) dst[r * NP + n + i] = r < nr && n + i < states ? (float)v[i] : 0.f;
    }
};
// LDS of one wave: what its lanes wrote is there for all of them (the hardware keeps a wave's LDS accesses in order; this keeps the compiler's)
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Where a lane works
template <int L, int NS> struct Lane {
    int lane, wave, j, c, n0, nn; bool ok, full; int g;
    __device__ __forceinline__ Lane(const ScanK& k, int waves, int blk) {
        lane = threadIdx.x & 63; wave = uniform(threadIdx.x >> 6);
        j = lane % L;
        g = blk / k.nblk;
        const int cw = 64 / L, cb = (blk - g * k.nblk) * waves * cw + wave * cw + lane / L;
        ok = cb < k.cg;
        c = g * k.cg + min(cb, k.cg - 1);
        n0 = j * NS;
        nn = max(0, min(NS, k.a.states - n0));
        full = k.a.states == L * NS;
    }
};
// a lane's states of a channel at p; `full` (the same in all lanes): none lacks any, so nothing waits for the answer of a branch
template <int NS> __device__ __forceinline__ void load_state(const float* p, float (&h)[NS], int nn, bool full) {
    if (full) load_vec<float, NS>(p, h); else load_some<float, NS>(p, h, nn);
}
template <int NS> __device__ __forceinline__ void store_state(float* p, const float (&h)[NS], int nn, bool full) {
    if (full) store_vec<float, NS>(p, h); else store_some<float, NS>(p, h, nn);
}

// Which register layout serves a number of states.  Four states a lane carry a row's fixed costs better than two: 64 x 128 x 1024 bf16, 32 states 94 us by
// 8 lanes of four, 140 by 16 of two (training 398 and 556).
#define SCAN_LAYOUT(T, states, F, ...) \
    ((states) <= 8 ? F<T, 4, 2>(__VA_ARGS__) : (states) <= 16 ? F<T, 4, 4>(__VA_ARGS__) : (states) <= 32 ? F<T, 8, 4>(__VA_ARGS__) : F<T, 16, 4>(__VA_ARGS__))
static inline int scan_lanes(int states) { return states <= 16 ? 4 : states <= 32 ? 8 : 16; }
static inline int scan_padded(int states) { return states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }
int scan_setup(const char* who, const vc_scan_args* a, int waves, int64_t run_waves, double margin, ScanK* k);
int64_t scan_edge_floats(const ScanK& k);                        // of edge, sum_delta and cut
void scan_edge_place(ScanK* k, float* work);
// What enters run `item` from the runs before it (behind it where !FORWARD).  Up to CARRY_ITEMS runs every wave goes through them itself, which saves a
// launch; more are gone through once for all by scan_carry, which puts what enters a run in the place of what it hands on.  1 x 8192 x 1024 (64 runs)
// 102 us by the waves, 100 by scan_carry; 1 x 512 x 1024 (33) 17 and 18; 8 x 128 x 1024 training (up to 32) 70 and 74.
constexpr int CARRY_ITEMS = 32;
// exp2(p) h + e, or e where nothing is handed on.  In two halves: the factor of a whole run may leave the range of fp32 where its product with h does not
// (frame by frame it would not either), and a state of zero stays one under any factor.  A factor that is only too small for fp32 is 2^-252 in place of 0, which
// leaves nothing of a finite state and an infinite one as it is (0 would make it no number).
__device__ __forceinline__ float carried(float p, float h, float e, int cut) {
    const float f = fmaxf(exp2_fast(0.5f * p), p >= -3.4e38f ? 0x1p-126f : 0.f);             // (where p is no number, e is none)
    return cut || h == 0.f ? e : fmaf(f * h, f, e);
}
int scan_carry(const ScanK& k, bool forward, hipStream_t s);
template <int NS, bool FORWARD> __device__ __forceinline__ void carry_in(const ScanK& k, int item, int c, int n0, int nn, bool full, const float (&A2)[NS], float (&h)[NS]) {
    constexpr int AT_ONCE = 8;                                   // runs whose loads are on their way together: the chain itself is one multiply-add a run
    const vc_scan_args& a = k.a;
    if (k.once) {
        load_state<NS>(k.edge + ((int64_t)item * a.cols + c) * a.states + n0, h, nn, full);
        return;
    }
    const int n = FORWARD ? item : k.items - 1 - item;           // runs to go through, the farthest first
    for (int i0 = 0; i0 < n; i0 += AT_ONCE) {
        float e[AT_ONCE][NS], sd[AT_ONCE]; int cut[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int at = min(i0 + i, n - 1), r = FORWARD ? at : k.items - 1 - at;
            load_state<NS>(k.edge + ((int64_t)r * a.cols + c) * a.states + n0, e[i], nn, full);
            sd[i] = k.sum_delta[(int64_t)r * a.cols + c];
            cut[i] = k.cut[r];
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (i0 + i >= n) break;
#pragma unroll
            for (int j = 0; j < NS; ++j) h[j] = carried(A2[j] * sd[i], h[j], e[i][j], cut[i]);
        }
    }
}
