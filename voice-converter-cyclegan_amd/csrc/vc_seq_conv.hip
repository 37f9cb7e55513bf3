// vc_seq_conv.hip -- short causal convolution along the rows, one filter per channel: prompts, gradient, single frames.
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k];  y = p sigmoid(p) or p
#include "vc_seq.h"

struct ConvArgs { vc_conv1d_args a; SeqMap m; };

// the utterance row r lies in: the last s with begin(s) <= r whose rows are not none; n_seqs where r lies behind the last utterance
__device__ __forceinline__ int seq_of(const SeqMap& m, int r) {
    if (!m.off) return r / m.len;
    if (r >= seq_tail(m)) return m.n_seqs;
    int lo = 0, hi = m.n_seqs - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (seq_begin(m, mid) <= r) lo = mid; else hi = mid - 1; }
    return lo;
}
// frame t (counted from the utterance's first row b) of channel c: the utterance's own, or an earlier one from the initial state
template <class T> __device__ __forceinline__ float frame(const vc_conv1d_args& a, int s, int b, int t, int c) {
    if (t >= 0) return (float)((const T*)a.x)[(int64_t)(b + t) * a.x_ld + c];
    return a.initial ? (float)((const T*)a.initial)[((int64_t)s * (a.taps - 1) + (a.taps - 1 + t)) * a.cols + c] : 0.f;
}
template <class T> __device__ __forceinline__ float pre(const vc_conv1d_args& a, int s, int b, int t, int c) {
    float p = a.bias ? a.bias[c] : 0.f;
    for (int k = 0; k < a.taps; ++k) p += a.w[k * a.cols + c] * frame<T>(a, s, b, t - (a.taps - 1) + k, c);
    return p;
}
// gradient of the pre-activation of frame t
template <class T> __device__ __forceinline__ float dpre(const vc_conv1d_args& a, int s, int b, int t, int c) {
    const float g = (float)((const T*)a.dy)[(int64_t)(b + t) * a.dy_ld + c];
    if (!a.silu) return g;
    const float p = pre<T>(a, s, b, t, c), sg = sigmoid_acc(p);
    return g * sg * (1.f + p * (1.f - sg));
}
template <class T> __global__ __launch_bounds__(256) void conv1d_fwd_kernel(const ConvArgs k) {
    const vc_conv1d_args& a = k.a;
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    for (int r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const int s = seq_of(k.m, r);
        if (s == k.m.n_seqs) { if (a.zero_tail) ((T*)a.y)[(int64_t)r * a.y_ld + c] = (T)0.f; continue; }
        const int b = seq_begin(k.m, s);
        const float p = pre<T>(a, s, b, r - b, c);
        ((T*)a.y)[(int64_t)r * a.y_ld + c] = (T)(a.silu ? p * sigmoid_acc(p) : p);
    }
    if (a.final_state)
        for (int s = blockIdx.y; s < k.m.n_seqs; s += gridDim.y) {
            const int b = seq_begin(k.m, s), e = seq_end(k.m, s, b);
            for (int i = 0; i < a.taps - 1; ++i)
                ((T*)a.final_state)[((int64_t)s * (a.taps - 1) + i) * a.cols + c] = (T)frame<T>(a, s, b, e - b - (a.taps - 1) + i, c);
        }
}
// gradient of frame t of the utterance (t < 0: of the initial state's)
template <class T> __device__ __forceinline__ float dframe(const vc_conv1d_args& a, int s, int b, int n, int t, int c) {
    float d = 0.f;
    for (int k = 0; k < a.taps; ++k) { const int o = t + (a.taps - 1) - k; if (o >= 0 && o < n) d += a.w[k * a.cols + c] * dpre<T>(a, s, b, o, c); }
    if (a.dfinal && t >= n - (a.taps - 1)) d += (float)((const T*)a.dfinal)[((int64_t)s * (a.taps - 1) + t - (n - (a.taps - 1))) * a.cols + c];
    return d;
}
template <class T> __global__ __launch_bounds__(256) void conv1d_bwd_kernel(const ConvArgs k) {
    const vc_conv1d_args& a = k.a;
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    if (a.dx)
        for (int r = blockIdx.y; r < a.rows; r += gridDim.y) {
            const int s = seq_of(k.m, r);
            if (s == k.m.n_seqs) { if (a.zero_tail) ((T*)a.dx)[(int64_t)r * a.dx_ld + c] = (T)0.f; continue; }
            const int b = seq_begin(k.m, s), e = seq_end(k.m, s, b);
            ((T*)a.dx)[(int64_t)r * a.dx_ld + c] = (T)dframe<T>(a, s, b, e - b, r - b, c);
        }
    if (a.dinitial)
        for (int s = blockIdx.y; s < k.m.n_seqs; s += gridDim.y) {
            const int b = seq_begin(k.m, s), e = seq_end(k.m, s, b);
            for (int i = 0; i < a.taps - 1; ++i)
                ((T*)a.dinitial)[((int64_t)s * (a.taps - 1) + i) * a.cols + c] = (T)dframe<T>(a, s, b, e - b, i - (a.taps - 1), c);
        }
}
template <class T> __global__ __launch_bounds__(64) void conv1d_dw_kernel(const ConvArgs k) {
    const vc_conv1d_args& a = k.a;
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= a.cols) return;
    float dw[8] = {}, db = 0.f;
    for (int s = 0; s < k.m.n_seqs; ++s) {
        const int b = seq_begin(k.m, s), n = seq_end(k.m, s, b) - b;
        for (int t = 0; t < n; ++t) {
            const float g = dpre<T>(a, s, b, t, c);
            db += g;
#pragma unroll
            for (int j = 0; j < 8; ++j) if (j < a.taps) dw[j] += g * frame<T>(a, s, b, t - (a.taps - 1) + j, c);
        }
    }
    if (a.dbias) a.dbias[c] = db;
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < a.taps && a.dw) a.dw[j * a.cols + c] = dw[j];
}
struct ConvStepArgs {
    const void* x; void* state; const int* slots; const float *w, *bias; void* y;
    int64_t x_ld, y_ld; int rows, n_slots, cols, taps, silu;
};
// The slot row r works on, -1 where it is padding: outside the pool, or named by an earlier row of this call.  Every thread of the block calls it.
__device__ __forceinline__ int claim_slot(const int* slots, int r, int n_slots) {
    const int mine = slots ? slots[r] : r;
    int taken = mine < 0 || mine >= n_slots;
    if (slots)
        for (int i = threadIdx.x; i < r; i += blockDim.x) taken |= slots[i] == mine;
    return __syncthreads_or(taken) ? -1 : mine;
}
template <class T> __global__ __launch_bounds__(256) void conv1d_step_kernel(const ConvStepArgs a) {
    const int r = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    const int slot = claim_slot(a.slots, r, a.n_slots);
    if (c >= a.cols) return;
    T* y = (T*)a.y + (int64_t)r * a.y_ld + c;
    if (slot < 0) { *y = (T)0.f; return; }
    T* st = (T*)a.state + (int64_t)slot * (a.taps - 1) * a.cols + c;
    const T x = ((const T*)a.x)[(int64_t)r * a.x_ld + c];
    float p = (a.bias ? a.bias[c] : 0.f);
    for (int k = 0; k < a.taps - 1; ++k) {
        const T v = st[(int64_t)k * a.cols];
        p += a.w[k * a.cols + c] * (float)v;
        if (k) st[(int64_t)(k - 1) * a.cols] = v;
    }
    p += a.w[(a.taps - 1) * a.cols + c] * (float)x;
    st[(int64_t)(a.taps - 2) * a.cols] = x;
    *y = (T)(a.silu ? p * sigmoid_acc(p) : p);
}

static int check_conv1d(const char* who, const vc_conv1d_args* a, ConvArgs* k) {
    VC_ARG(a, "%s: null pointer", who);
    VC_ARG(seq_type_ok(a->type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(a->taps >= 2 && a->taps <= 8, "%s: 2 to 8 taps, got %d", who, a->taps);
    VC_ARG(a->rows >= 0 && a->rows < (1LL << 31) - (1 << 16) && a->cols > 0 && a->n_seqs > 0, "%s: bad sizes (rows %lld, cols %d, n_seqs %d)", who, (long long)a->rows, a->cols, a->n_seqs);
    VC_ARG(a->offsets || a->rows % a->n_seqs == 0, "%s: without offsets the rows divide into n_seqs equal utterances", who);
    k->a = *a;
    k->m = SeqMap{a->offsets, (int)a->rows, a->n_seqs, (int)(a->rows / a->n_seqs)};
    return 0;
}
template <class T> static int conv1d_fwd(const ConvArgs& k, hipStream_t s) {
    const int n = (int)std::max<int64_t>(k.a.rows, k.a.n_seqs);
    hipLaunchKernelGGL((conv1d_fwd_kernel<T>), dim3((k.a.cols + 255) / 256, std::min(n, 32768)), dim3(256), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int conv1d_bwd(const ConvArgs& k, hipStream_t s) {
    const int n = (int)std::max<int64_t>(k.a.rows, k.a.n_seqs);
    hipLaunchKernelGGL((conv1d_bwd_kernel<T>), dim3((k.a.cols + 255) / 256, std::min(n, 32768)), dim3(256), 0, s, k);
    if (k.a.dw || k.a.dbias) hipLaunchKernelGGL((conv1d_dw_kernel<T>), dim3((k.a.cols + 63) / 64), dim3(64), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int conv1d_step(const ConvStepArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((conv1d_step_kernel<T>), dim3((a.cols + 255) / 256, a.rows), dim3(256), 0, s, a);
    VC_HIP(hipGetLastError());
    return 0;
}
extern "C" int vc_causal_conv1d_fwd(const vc_conv1d_args* a, void* stream) {
    ConvArgs k; VC_CHECK(check_conv1d("vc_causal_conv1d_fwd", a, &k));
    VC_ARG(a->w && (a->rows == 0 || (a->x && a->y)), "vc_causal_conv1d_fwd: null pointer");
    VC_ARG(!a->final_state || a->final_state != a->initial, "vc_causal_conv1d_fwd: final_state may not be initial");
    if (a->rows == 0 && !a->final_state) return 0;
    return SEQ_TYPES(a->type, conv1d_fwd, k, (hipStream_t)stream);
}
extern "C" int64_t vc_causal_conv1d_bwd_work(const vc_conv1d_args* a) { return 0; }
extern "C" int vc_causal_conv1d_bwd(const vc_conv1d_args* a, void* stream) {
    ConvArgs k; VC_CHECK(check_conv1d("vc_causal_conv1d_bwd", a, &k));
    VC_ARG(a->w && (a->rows == 0 || (a->x && a->dy)), "vc_causal_conv1d_bwd: null pointer");
    return SEQ_TYPES(a->type, conv1d_bwd, k, (hipStream_t)stream);
}
extern "C" int vc_causal_conv1d_step(const void* x, int64_t x_ld, void* state, const int32_t* slots, const float* w, const float* bias,
                                     void* y, int64_t y_ld, int rows, int n_slots, int cols, int taps, int type, int silu, void* stream) {
    VC_ARG(seq_type_ok(type), "vc_causal_conv1d_step: type must be VC_F32, VC_BF16 or VC_F16");
    VC_ARG(taps >= 2 && taps <= 8, "vc_causal_conv1d_step: 2 to 8 taps, got %d", taps);
    VC_ARG(rows >= 0 && rows <= 65535 && n_slots > 0 && cols > 0, "vc_causal_conv1d_step: bad sizes (rows %d, n_slots %d, cols %d)", rows, n_slots, cols);
    VC_ARG(slots || rows <= n_slots, "vc_causal_conv1d_step: %d rows without slots, and %d slots", rows, n_slots);
    if (rows == 0) return 0;
    VC_ARG(x && state && w && y, "vc_causal_conv1d_step: null pointer");
    const ConvStepArgs a{x, state, slots, w, bias, y, x_ld, y_ld, rows, n_slots, cols, taps, silu};
    return SEQ_TYPES(type, conv1d_step, a, (hipStream_t)stream);
}
