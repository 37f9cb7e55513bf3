// vc_seq.h -- what the translation units of the sequence operators share (vc_seq_norm.hip, vc_seq_conv.hip, vc_seq_scan.hip, vc_seq_scan_bwd.hip):
// element types, utterance offsets, lane exchanges.
#pragma once
#include "vc_host.h"
#include "vc_device_util.h"
#include <algorithm>
#include <type_traits>

// F<T>(arguments) for the element type that `type` names
#define SEQ_TYPES(type, F, ...) ((type) == VC_F32 ? F<float>(__VA_ARGS__) : (type) == VC_BF16 ? F<__bf16>(__VA_ARGS__) : F<_Float16>(__VA_ARGS__))
static inline int seq_esize(int type) { return type == VC_F32 ? 4 : 2; }
// Channels of a call: column indexes of the norm and of the convolution, and what they step over, then stay within 31 bits
constexpr int64_t NORM_COLS = 1 << 28, SEQ_COLS = 1 << 24;
static inline bool seq_type_ok(int type) { return type == VC_F32 || type == VC_BF16 || type == VC_F16; }

// V elements in one access at any address the element type itself allows: gfx950 takes 16-byte global accesses at any alignment, so odd
// channel counts and row strides need no second path
template <class T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };
template <class T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
    const Pack<T, V> q = *(const Pack<T, V>*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)q.v[i];
}
template <class T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
    Pack<T, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = (T)f[i];
    *(Pack<T, V>*)p = q;
}
// the first n of V elements (the rest reads as zero)
template <class T, int V> __device__ __forceinline__ void load_some(const T* p, float (&f)[V], int n) {
    if (n >= V) { load_vec<T, V>(p, f); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < n ? (float)p[i] : 0.f;
}
template <class T, int V> __device__ __forceinline__ void store_some(T* p, const float (&f)[V], int n) {
    if (n >= V) { store_vec<T, V>(p, f); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < n) p[i] = (T)f[i];
}

// Stores that the L2s are not to keep (non-temporal), for calls whose output is larger than what the next kernel would find there of it anyway: the lines
// then do not push out what is still to be read.  8192 x 2048 bf16 convolution with its gradient 46 us without, 41 with; norm of 16384 x 2048 and the product
// behind it 111 and 86, of 8192 x 1024 34 and 32, of 4096 x 1024 24 and 24, of 2048 x 1024 17 and 18.
constexpr int64_t STREAM_BYTES = 8 << 20;                        // of one tensor
typedef unsigned Quad __attribute__((ext_vector_type(4), aligned(2)));
template <class T, int V> __device__ __forceinline__ void store_out(T* p, const float (&f)[V], int n, bool past) {
    Pack<T, V> q;
    if constexpr (sizeof(q) % 16 == 0) {
        if (past && n >= V) {
            struct Quads { Quad w[sizeof(q) / 16]; };
#pragma unroll
            for (int i = 0; i < V; ++i) q.v[i] = (T)f[i];
            const Quads w = __builtin_bit_cast(Quads, q);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(q) / 16); ++i) __builtin_nontemporal_store(w.w[i], (Quad*)p + i);
            return;
        }
    }
    store_some<T, V>(p, f, n);
}

// ... and such loads, where a thread takes a vector in one access (two would fetch their line twice) and rows share no line.  Only where a pass reads
// LOAD_BYTES or more in all: of fewer the last level of cache may still hold much.  Norm kernels of 1024 or 2048 columns on three sets of tensors in turn, us
// without and with, by what a pass reads: forward of bf16 rows 64 MiB 24.3 and 24.9, 80 MiB 29.4 and 30.0, 88 MiB 39.8 and 32.5, 128 MiB 54.8 and 46.1; of fp32
// rows 64 MiB 21.3 and 24.2, 80 MiB 26.0 and 29.6, 88 MiB 33.1 and 32.3, 128 MiB 48.7 and 45.3; to 8 bits 64 MiB 32.2 and 32.5 (2048 x 8192: 38.1 and 41.2), 80 MiB
// 41.4 and 38.1, 96 MiB 48.9 and 45.1; gradient 60 MiB 26.1 and 25.5, 84 MiB 37.4 and 33.3, 96 MiB 40.8 and 34.0, fp32 33.6 and 34.7 (1024 columns 33.3 and 29.9),
// 192 MiB 75.7 and 61.0, fp32 56.3 and 56.1.  Between a kernel that has just written the input and one that reads the result such loads win at all sizes
// (16-bit rows up to 10 %, fp32 1 %); below the border they are left out for the calls that find their inputs in the cache.
constexpr int64_t LOAD_BYTES = 88 << 20;                         // of all tensors that a pass reads
template <class T, int V> __device__ __forceinline__ void load_in(const T* p, float (&f)[V], int n, bool past) {
    if constexpr (V * sizeof(T) == 16) {
        if (past && n >= V) {
            const Pack<T, V> q = __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load((const Quad*)p));
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (float)q.v[i];
            return;
        }
    }
    load_some<T, V>(p, f, n);
}

// The utterances of one call.  begin / end clamp into [0, rows], whatever the device array holds.
struct SeqMap { const int* off; int rows, n_seqs, len; };
__device__ __forceinline__ int seq_begin(const SeqMap& m, int s) { return m.off ? min(max(m.off[s], 0), m.rows) : s * m.len; }
__device__ __forceinline__ int seq_end(const SeqMap& m, int s, int begin) { return m.off ? max(seq_begin(m, s + 1), begin) : begin + m.len; }
// the utterances begin here (rows ahead of it belong to none), and rows behind the last one here
__device__ __forceinline__ int seq_head(const SeqMap& m) { return m.off ? seq_begin(m, 0) : 0; }
__device__ __forceinline__ int seq_tail(const SeqMap& m) { return m.off ? seq_begin(m, m.n_seqs) : m.rows; }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f, LN2_REST = -1.90465429995776804525e-9f;       // log 2 = LN2 + LN2_REST
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// e^v for -128 <= v <= 88.72 (0 where it leaves fp32 downwards): 2^t of t = v log2 e as it is rounded, and what that leaves out put back, e^c = 1 + c with
// c = v - t log 2: the exponential alone would be off by |v| 2^-24 of itself
__device__ __forceinline__ float exp_acc(float v) {
    const float t = v * LOG2E, c = fmaf(t, -LN2_REST, fmaf(t, -LN2, v)), e = exp2_fast(t);
    return fmaf(e, c, e);
}
// 1 / (1 + e^-x) for activations of type T.  fp32: 6 roundings of 2^-24 relative to itself, the exponential 2 and its correction, 1 + e, the reciprocal 2.
// Below -87.34, where it leaves the normal numbers, it is 0 (the reciprocal is flushed; bounded at -88.72 so that e stays finite), far above 1; of a NaN it is
// a number, but everything here multiplies it by x.
// 16-bit activations: without the correction, off by |x| 2^-24 of itself for negative x; what it goes into is rounded by 2^-9 or 2^-12 (and parameter
// gradients add it to terms that are not that small).  8192 x 2048 bf16 convolution and gradient 41 us so, 46 with it; 9001 x 1000 fp32 17.6 without, 18.1 with.
template <class T> __device__ __forceinline__ float sigmoid(float x) {
    if constexpr (sizeof(T) == 4) return __builtin_amdgcn_rcpf(1.f + exp_acc(-__builtin_amdgcn_fmed3f(x, -88.72f, 128.f)));
    else return __builtin_amdgcn_rcpf(1.f + __expf(-x));
}
// Single-frame calls.  The slot row r names; whether it is padding: a slot outside the pool, or one that an earlier row of the call names.  A wave looks
// through the earlier rows itself (no barrier); MAX_SLOT_ROWS bounds how many there are.
constexpr int MAX_SLOT_ROWS = 4096;
__device__ __forceinline__ bool slot_is_padding(const int* slots, int r, int mine, int n_slots) {
    bool taken = mine < 0 || mine >= n_slots;
    if (slots) {
#pragma unroll 4
        for (int i = threadIdx.x & 63; i < r; i += 64) taken |= slots[i] == mine;
    }
    return __any(taken);
}

// dst[i] = sum over `parts` rows of part[parts][n], in order; columns [0, n0) go to dst0, the others to dst1 (either may be null).  vc_seq_norm.hip
int seq_sum_parts(const float* part, int parts, int64_t n, float* dst0, int64_t n0, float* dst1, hipStream_t s);
