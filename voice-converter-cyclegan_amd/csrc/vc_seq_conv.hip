// vc_seq_conv.hip -- short causal convolution along the rows, one filter per channel: prompts, gradient, single frames.
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k];  y = p sigmoid(p) or p
//   g = dy * (p sigmoid(p))';  dx[u] = sum_k w[k] g[u + (K-1) - k];  dw[k] = sum_t g[t] x[t - (K-1) + k];  dbias = sum_t g[t]
// Bound by HBM.  A thread walks a run of rows for one 16-byte vector of channels with the last K frames in registers, so a row is fetched once,
// apart from the K - 1 frames ahead of a run.
#include "vc_seq.h"

struct ConvArgs { vc_conv1d_args a; SeqMap m; int v, cv, cvb, runs; float* part; };     // v channels a thread, cv such vectors, cvb of them next to each other

// the utterance row r lies in: the last s with begin(s) <= r; n_seqs where r lies behind the last utterance
__device__ __forceinline__ int seq_of(const SeqMap& m, int r) {
    if (!m.off) return r / m.len;
    if (r >= seq_tail(m)) return m.n_seqs;
    int lo = 0, hi = m.n_seqs - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (seq_begin(m, mid) <= r) lo = mid; else hi = mid - 1; }
    return lo;
}
// V channels of frame t (counted from the utterance's first row b): the utterance's own, or an earlier one from the initial state
template <class T, int V> __device__ __forceinline__ void frame(const vc_conv1d_args& a, int s, int b, int t, int c, float (&f)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = 0.f;
    if (t >= 0) load_vec<T, V>((const T*)a.x + (int64_t)(b + t) * a.x_ld + c, f);
    else if (a.initial) load_vec<T, V>((const T*)a.initial + ((int64_t)s * (a.taps - 1) + (a.taps - 1 + t)) * a.cols + c, f);
}
template <class T, int K, int V> struct Filter {
    float w[K][V], b[V];
    __device__ __forceinline__ Filter(const vc_conv1d_args& a, int c) {
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] = 0.f;
        if (a.bias) load_vec<float, V>(a.bias + c, b);
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < V; ++e) w[k][e] = 0.f;
            load_vec<float, V>(a.w + (int64_t)k * a.cols + c, w[k]);
        }
    }
};
// A block's threads: cvb vectors of channels (a power of two) next to each other, 256 / cvb runs of rows
// Rows of a run, and rows whose loads are issued together while as many are worked on.  8192 x 2048 bf16, 4 taps, forward and backward: 46.5 us
// with (8, 16; 4, 2); 49.6 with (16, 16; 4, 4), 51.9 with (16, 16; 2, 2), 47.4 with (32, 32; 4, 4), which gives small calls too few threads.
constexpr int FWD_RUN = 8, BWD_RUN = 16, FWD_AHEAD = 4, BWD_AHEAD = 2;
constexpr int BWD_V = 4;                                         // channels of a thread of the gradient
constexpr int FWD_WIDE = 32, BWD_WIDE = 64;                      // most vectors of channels next to each other in a block
struct Place { int c, run; bool ok; };
__device__ __forceinline__ Place place(const ConvArgs& k, int V) {
    const int blocks = (k.cv + k.cvb - 1) / k.cvb;
    Place p;
    const int v = (int)(blockIdx.x % blocks) * k.cvb + threadIdx.x % k.cvb;
    p.run = (int)(blockIdx.x / blocks) * (256 / k.cvb) + threadIdx.x / k.cvb;
    // the last vector ends with the last channel: where V does not divide the channels it works out some of its neighbour's once more, to the same
    // values, and no access has to ask how many channels are left (fewer than V of them: V = 1)
    p.c = min(v * V, k.a.cols - V); p.ok = v < k.cv;
    return p;
}

// V elements as they came: 16-bit ones two to a register
template <class T, int V> struct Raw {
    static constexpr int N = (V * (int)sizeof(T) + 3) / 4;
    unsigned w[N];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V * sizeof(T) % 4 != 0) w[0] = __builtin_bit_cast(unsigned short, *p);
        else {
            struct __attribute__((packed, aligned(sizeof(T)))) W { unsigned v[N]; };
            const W q = *(const W*)p;
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = q.v[i];
        }
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (sizeof(T) == 4) f[i] = __builtin_bit_cast(float, w[i]);
            else f[i] = (float)__builtin_bit_cast(T, (unsigned short)(w[i / 2] >> (16 * (i % 2))));
        }
    }
};
template <class T, int K, int V> __global__ __launch_bounds__(256) void conv1d_fwd_kernel(const ConvArgs k) {
    const vc_conv1d_args& a = k.a;
    const Place p = place(k, V);
    if (!p.ok) return;
    if (p.run >= k.runs) {                                       // behind the runs: one utterance's last K - 1 frames
        const int s = p.run - k.runs;
        if (!a.final_state || s >= k.m.n_seqs) return;
        const int b = seq_begin(k.m, s), e = seq_end(k.m, s, b);
#pragma unroll
        for (int i = 0; i < K - 1; ++i) {
            float f[V];
            frame<T, V>(a, s, b, e - b - (K - 1) + i, p.c, f);
            store_vec<T, V>((T*)a.final_state + ((int64_t)s * (K - 1) + i) * a.cols + p.c, f);
        }
        return;
    }
    const Filter<T, K, V> w(a, p.c);
    int r = p.run * FWD_RUN;
    const int r1 = min(r + FWD_RUN, k.m.rows);
    const T* x = (const T*)a.x + p.c;
    T* y = (T*)a.y + p.c;
    for (int s = seq_of(k.m, r); r < r1; ++s) {
        if (s >= k.m.n_seqs) {                                   // rows behind the last utterance
            float f[V] = {};
            if (a.zero_tail) for (; r < r1; ++r) store_vec<T, V>(y + (int64_t)r * a.y_ld, f);
            return;
        }
        const int b = seq_begin(k.m, s), hi = min(seq_end(k.m, s, b), r1);
        if (r >= hi) continue;                                   // an empty utterance
        float win[K][V];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) frame<T, V>(a, s, b, r - b - (K - 1) + i, p.c, win[i]);
        auto step = [&](const float (&f)[V]) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                win[K - 1][e] = f[e];
                float q = w.b[e];
#pragma unroll
                for (int i = 0; i < K; ++i) q = fmaf(w.w[i][e], win[i][e], q);
                o[e] = a.silu ? q * sigmoid_acc(q) : q;
#pragma unroll
                for (int i = 0; i < K - 1; ++i) win[i][e] = win[i + 1][e];
            }
            store_vec<T, V>(y + (int64_t)r * a.y_ld, o);
            ++r;
        };
        // FWD_AHEAD rows are worked on while the next are on their way; rows past the end read the last one and are not used
        Raw<T, V> next[FWD_AHEAD];
        auto fetch = [&](int at) {
#pragma unroll
            for (int i = 0; i < FWD_AHEAD; ++i) next[i].load(x + (int64_t)min(at + i, hi - 1) * a.x_ld);
        };
        fetch(r);
        while (r < hi) {
            Raw<T, V> now[FWD_AHEAD];
#pragma unroll
            for (int i = 0; i < FWD_AHEAD; ++i) now[i] = next[i];
            if (r + FWD_AHEAD < hi) fetch(r + FWD_AHEAD);
#pragma unroll
            for (int i = 0; i < FWD_AHEAD; ++i) {
                if (r >= hi) break;
                float f[V];
                now[i].get(f);
                step(f);
            }
        }
    }
}

// g of one frame, from the K frames it looks at
template <int K, int V> __device__ __forceinline__ void pre_gradient(const float (&win)[K][V], const float (&w)[K][V], const float (&b)[V], bool silu, float (&g)[V]) {
    if (!silu) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float q = b[e];
#pragma unroll
        for (int i = 0; i < K; ++i) q = fmaf(w[i][e], win[i][e], q);
        const float sg = sigmoid_acc(q);
        g[e] *= sg * fmaf(q, 1.f - sg, 1.f);
    }
}
// A run's dx needs the K - 1 frames' g behind it as well: they are worked out again there.  dx of a frame gathers in a register ring while the
// frames that look at it go by.
// Four channels a thread: eight would fill the registers (filter, window, ring and its share of dw are K vectors each) and leave too few waves to wait with.
template <class T, int K, int V> __global__ __launch_bounds__(256) void conv1d_bwd_kernel(const ConvArgs k) {
    __shared__ float red[256 * V];
    const vc_conv1d_args& a = k.a;
    const Place p = place(k, V);
    float dw[K][V] = {}, db[V] = {};
    if (p.ok && p.run < k.runs) {
        const Filter<T, K, V> w(a, p.c);
        int r = p.run * BWD_RUN;
        const int r1 = min(r + BWD_RUN, k.m.rows);
        const T *x = (const T*)a.x + p.c, *dy = (const T*)a.dy + p.c;
        T* dx = a.dx ? (T*)a.dx + p.c : nullptr;
        for (int s = seq_of(k.m, r); r < r1; ++s) {
            if (s >= k.m.n_seqs) {
                float f[V] = {};
                if (a.zero_tail && dx) for (; r < r1; ++r) store_vec<T, V>(dx + (int64_t)r * a.dx_ld, f);
                break;
            }
            const int b = seq_begin(k.m, s), end = seq_end(k.m, s, b), lo = r, hi = min(end, r1);
            if (lo >= hi) continue;
            float win[K][V], ring[K][V] = {};                    // ring[i]: dx of frame r - (K-1) + i so far
#pragma unroll
            for (int i = 0; i < K - 1; ++i) frame<T, V>(a, s, b, lo - b - (K - 1) + i, p.c, win[i]);
            auto emit = [&](int at, const float (&d)[V]) {       // row `at` has all but its share of the final state's gradient
                if (!dx || at < lo || at >= hi) return;
                float o[V] = {};
                if (a.dfinal && at >= end - (K - 1))
                    load_vec<T, V>((const T*)a.dfinal + ((int64_t)s * (K - 1) + at - (end - (K - 1))) * a.cols + p.c, o);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += d[e];
                store_vec<T, V>(dx + (int64_t)at * a.dx_ld, o);
            };
            auto step = [&](const float (&f)[V], float (&g)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e) win[K - 1][e] = f[e];
                pre_gradient<K, V>(win, w.w, w.b, a.silu, g);
                if (r < hi) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        db[e] += g[e];
#pragma unroll
                        for (int i = 0; i < K; ++i) dw[i][e] = fmaf(g[e], win[i][e], dw[i][e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e)
#pragma unroll
                    for (int i = 0; i < K; ++i) ring[i][e] = fmaf(w.w[i][e], g[e], ring[i][e]);
                emit(r - (K - 1), ring[0]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
#pragma unroll
                    for (int i = 0; i < K - 1; ++i) { win[i][e] = win[i + 1][e]; ring[i][e] = ring[i + 1][e]; }
                    ring[K - 1][e] = 0.f;
                }
                ++r;
            };
            const int stop = min(end, hi + (dx ? K - 1 : 0));
            // BWD_AHEAD rows are worked on while the next are on their way; rows past the end read the last one and are not used
            Raw<T, V> xn[BWD_AHEAD], gn[BWD_AHEAD];
            auto fetch = [&](int at) {
#pragma unroll
                for (int i = 0; i < BWD_AHEAD; ++i) {
                    const int64_t row = min(at + i, stop - 1);
                    xn[i].load(x + row * a.x_ld); gn[i].load(dy + row * a.dy_ld);
                }
            };
            fetch(r);
            while (r < stop) {
                Raw<T, V> xc[BWD_AHEAD], gc[BWD_AHEAD];
#pragma unroll
                for (int i = 0; i < BWD_AHEAD; ++i) { xc[i] = xn[i]; gc[i] = gn[i]; }
                if (r + BWD_AHEAD < stop) fetch(r + BWD_AHEAD);
#pragma unroll
                for (int i = 0; i < BWD_AHEAD; ++i) {
                    if (r >= stop) break;
                    float f[V], g[V];
                    xc[i].get(f); gc[i].get(g);
                    step(f, g);
                }
            }
#pragma unroll
            for (int i = 0; i < K - 1; ++i) emit(stop - (K - 1) + i, ring[i]);      // the utterance's last frames, nothing behind them
            r = hi;
        }
    } else if (p.ok && a.dinitial && p.run - k.runs < k.m.n_seqs) {
        const int s = p.run - k.runs;                            // gradient of the K - 1 frames ahead of one utterance
        const Filter<T, K, V> w(a, p.c);
        const int b = seq_begin(k.m, s), len = seq_end(k.m, s, b) - b;
        float win[K][V], ring[K - 1][V] = {};
#pragma unroll
        for (int i = 0; i < K - 1; ++i) frame<T, V>(a, s, b, i - (K - 1), p.c, win[i]);
#pragma unroll
        for (int t = 0; t < K - 1; ++t) {
            if (t >= len) continue;
            float g[V] = {};
            frame<T, V>(a, s, b, t, p.c, win[K - 1]);
            load_vec<T, V>((const T*)a.dy + (int64_t)(b + t) * a.dy_ld + p.c, g);
            pre_gradient<K, V>(win, w.w, w.b, a.silu, g);
#pragma unroll
            for (int i = 0; i < K - 1; ++i)                      // frame t's tap j looks at frame t - (K-1) + j = i - (K-1)
                if (i - t >= 0)
#pragma unroll
                    for (int e = 0; e < V; ++e) ring[i][e] = fmaf(w.w[i - t >= 0 ? i - t : 0][e], g[e], ring[i][e]);
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) win[i][e] = win[i + 1][e];
        }
#pragma unroll
        for (int i = 0; i < K - 1; ++i) {
            float o[V] = {};
            if (a.dfinal && i >= len) load_vec<T, V>((const T*)a.dfinal + ((int64_t)s * (K - 1) + i - len) * a.cols + p.c, o);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] += ring[i][e];
            store_vec<T, V>((T*)a.dinitial + ((int64_t)s * (K - 1) + i) * a.cols + p.c, o);
        }
    }
    if (!k.part) return;
    const int blocks = (k.cv + k.cvb - 1) / k.cvb, row = blockIdx.x / blocks;
    if (row * (256 / k.cvb) >= k.runs) return;                   // no run in this block
    float* part = k.part + (int64_t)row * (K + 1) * a.cols;
    auto combine = [&](const float (&v)[V], float* dst) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[e * 256 + threadIdx.x] = v[e];
        __syncthreads();
        if (threadIdx.x >= (unsigned)k.cvb || !p.ok) return;
        float s[V] = {};
        for (int i = threadIdx.x; i < 256; i += k.cvb)
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += red[e * 256 + i];
        store_vec<float, V>(dst + p.c, s);
    };
#pragma unroll
    for (int i = 0; i < K; ++i) combine(dw[i], part + (int64_t)i * a.cols);
    combine(db, part + (int64_t)K * a.cols);
}

struct ConvStepArgs {
    const void* x; void* state; const int* slots; const float *w, *bias; void* y;
    int64_t x_ld, y_ld; int rows, n_slots, cols, taps, silu;
};
template <class T> __global__ __launch_bounds__(256) void conv1d_step_kernel(const ConvStepArgs a) {
    const int r = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    const int mine = a.slots ? a.slots[r] : r, at = mine >= 0 && mine < a.n_slots ? mine : 0, cc = min(c, a.cols - 1);
    const T* from = (const T*)a.state + (int64_t)at * (a.taps - 1) * a.cols + cc;
    const T x = ((const T*)a.x)[(int64_t)r * a.x_ld + cc];
    T f[7];
    float p = a.bias ? a.bias[cc] : 0.f;
#pragma unroll
    for (int k = 0; k < 7; ++k) {
        if (k >= a.taps - 1) break;
        f[k] = from[(int64_t)k * a.cols];
        p = fmaf(a.w[(int64_t)k * a.cols + cc], (float)f[k], p);
    }
    p = fmaf(a.w[(int64_t)(a.taps - 1) * a.cols + cc], (float)x, p);
    const bool padding = slot_is_padding(a.slots, r, mine, a.n_slots);
    if (c >= a.cols) return;
    T* y = (T*)a.y + (int64_t)r * a.y_ld + c;
    if (padding) { *y = (T)0.f; return; }
    *y = (T)(a.silu ? p * sigmoid_acc(p) : p);
    T* to = (T*)a.state + (int64_t)mine * (a.taps - 1) * a.cols + c;
#pragma unroll
    for (int k = 0; k < 7; ++k) {
        if (k >= a.taps - 1) break;
        to[(int64_t)k * a.cols] = k < 6 && k + 1 < a.taps - 1 ? f[k + 1 < 7 ? k + 1 : 6] : x;
    }
}

static int check_conv1d(const char* who, const vc_conv1d_args* a, int v, int most, ConvArgs* k) {
    VC_ARG(a, "%s: null pointer", who);
    VC_ARG(seq_type_ok(a->type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(a->taps >= 2 && a->taps <= 8, "%s: 2 to 8 taps, got %d", who, a->taps);
    VC_ARG(a->rows >= 0 && a->rows < (1LL << 31) - (1 << 16) && a->cols > 0 && a->n_seqs > 0, "%s: bad sizes (rows %lld, cols %d, n_seqs %d)", who, (long long)a->rows, a->cols, a->n_seqs);
    VC_ARG(a->offsets || a->rows % a->n_seqs == 0, "%s: without offsets the rows divide into n_seqs equal utterances", who);
    k->a = *a;
    k->m = SeqMap{a->offsets, (int)a->rows, a->n_seqs, (int)(a->rows / a->n_seqs)};
    k->v = a->cols < v ? 1 : v;
    k->cv = (a->cols + k->v - 1) / k->v;
    for (k->cvb = 1; k->cvb < k->cv && k->cvb < most;) k->cvb *= 2;
    k->part = nullptr;
    return 0;
}
static int conv_grid(const char* who, const ConvArgs& k, bool seqs, unsigned* grid) {
    const int per = 256 / k.cvb;
    const int64_t g = (int64_t)((k.cv + k.cvb - 1) / k.cvb) * (((int64_t)k.runs + (seqs ? k.m.n_seqs : 0) + per - 1) / per);
    VC_ARG(g < (1LL << 31), "%s: too many rows and channels for one launch", who);
    *grid = (unsigned)g;
    return 0;
}
template <class T, int K> static int fwd_k(const ConvArgs& k, unsigned grid, hipStream_t s) {
    if (k.v == 1) hipLaunchKernelGGL((conv1d_fwd_kernel<T, K, 1>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((conv1d_fwd_kernel<T, K, 16 / (int)sizeof(T)>), dim3(grid), dim3(256), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T, int K> static int bwd_k(const ConvArgs& k, unsigned grid, hipStream_t s) {
    if (k.v == 1) hipLaunchKernelGGL((conv1d_bwd_kernel<T, K, 1>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((conv1d_bwd_kernel<T, K, BWD_V>), dim3(grid), dim3(256), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
#define CONV_TAPS(T, taps, F, ...) \
    ((taps) == 2 ? F<T, 2>(__VA_ARGS__) : (taps) == 3 ? F<T, 3>(__VA_ARGS__) : (taps) == 4 ? F<T, 4>(__VA_ARGS__) : (taps) == 5 ? F<T, 5>(__VA_ARGS__) : \
     (taps) == 6 ? F<T, 6>(__VA_ARGS__) : (taps) == 7 ? F<T, 7>(__VA_ARGS__) : F<T, 8>(__VA_ARGS__))
template <class T> static int conv1d_fwd(const ConvArgs& k, unsigned grid, hipStream_t s) { return CONV_TAPS(T, k.a.taps, fwd_k, k, grid, s); }
template <class T> static int conv1d_bwd(const ConvArgs& k, unsigned grid, hipStream_t s) { return CONV_TAPS(T, k.a.taps, bwd_k, k, grid, s); }
template <class T> static int conv1d_step(const ConvStepArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((conv1d_step_kernel<T>), dim3((a.cols + 255) / 256, a.rows), dim3(256), 0, s, a);
    VC_HIP(hipGetLastError());
    return 0;
}
extern "C" int vc_causal_conv1d_fwd(const vc_conv1d_args* a, void* stream) {
    VC_ARG(a, "vc_causal_conv1d_fwd: null pointer");
    ConvArgs k; VC_CHECK(check_conv1d("vc_causal_conv1d_fwd", a, a->type == VC_F32 ? 4 : 8, FWD_WIDE, &k));
    VC_ARG(a->w && (a->rows == 0 || (a->x && a->y)), "vc_causal_conv1d_fwd: null pointer");
    VC_ARG(!a->final_state || a->final_state != a->initial, "vc_causal_conv1d_fwd: final_state may not be initial");
    if (a->rows == 0 && !a->final_state) return 0;
    k.runs = (k.m.rows + FWD_RUN - 1) / FWD_RUN;
    unsigned grid; VC_CHECK(conv_grid("vc_causal_conv1d_fwd", k, a->final_state != nullptr, &grid));
    return SEQ_TYPES(a->type, conv1d_fwd, k, grid, (hipStream_t)stream);
}
// rows of `part`: one for each block's runs
static int conv_parts(const ConvArgs& k) { const int per = 256 / k.cvb; return (k.runs + per - 1) / per; }
extern "C" int64_t vc_causal_conv1d_bwd_work(const vc_conv1d_args* a) {
    ConvArgs k; if (check_conv1d("vc_causal_conv1d_bwd_work", a, BWD_V, BWD_WIDE, &k)) return VC_E_ARG;
    k.runs = (k.m.rows + BWD_RUN - 1) / BWD_RUN;
    return (int64_t)conv_parts(k) * (a->taps + 1) * a->cols;
}
extern "C" int vc_causal_conv1d_bwd(const vc_conv1d_args* a, void* stream) {
    ConvArgs k; VC_CHECK(check_conv1d("vc_causal_conv1d_bwd", a, BWD_V, BWD_WIDE, &k));
    VC_ARG(a->w && (a->rows == 0 || (a->x && a->dy)), "vc_causal_conv1d_bwd: null pointer");
    k.runs = (k.m.rows + BWD_RUN - 1) / BWD_RUN;
    const bool params = a->dw || a->dbias;
    const int64_t need = (int64_t)conv_parts(k) * (a->taps + 1) * a->cols;
    if (params && need && (!a->work || a->work_floats < need)) { vc_set_error("vc_causal_conv1d_bwd: work is too small (%lld floats needed)", (long long)need); return VC_E_NOMEM; }
    if (params) k.part = a->work;
    unsigned grid; VC_CHECK(conv_grid("vc_causal_conv1d_bwd", k, a->dinitial != nullptr, &grid));
    if (grid) VC_CHECK(SEQ_TYPES(a->type, conv1d_bwd, k, grid, (hipStream_t)stream));
    // no rows: no parts, and the sums are zeros
    return params ? seq_sum_parts(k.part, conv_parts(k), (int64_t)(a->taps + 1) * a->cols, a->dw, (int64_t)a->taps * a->cols, a->dbias, (hipStream_t)stream) : 0;
}
extern "C" int vc_causal_conv1d_step(const void* x, int64_t x_ld, void* state, const int32_t* slots, const float* w, const float* bias,
                                     void* y, int64_t y_ld, int rows, int n_slots, int cols, int taps, int type, int silu, void* stream) {
    VC_ARG(seq_type_ok(type), "vc_causal_conv1d_step: type must be VC_F32, VC_BF16 or VC_F16");
    VC_ARG(taps >= 2 && taps <= 8, "vc_causal_conv1d_step: 2 to 8 taps, got %d", taps);
    VC_ARG(rows >= 0 && rows <= 65535 && n_slots > 0 && cols > 0, "vc_causal_conv1d_step: bad sizes (rows %d, n_slots %d, cols %d)", rows, n_slots, cols);
    VC_ARG(slots || rows <= n_slots, "vc_causal_conv1d_step: %d rows without slots, and %d slots", rows, n_slots);
    VC_ARG(!slots || rows <= MAX_SLOT_ROWS, "vc_causal_conv1d_step: at most %d rows with slots, got %d", MAX_SLOT_ROWS, rows);
    if (rows == 0) return 0;
    VC_ARG(x && state && w && y, "vc_causal_conv1d_step: null pointer");
    const ConvStepArgs a{x, state, slots, w, bias, y, x_ld, y_ld, rows, n_slots, cols, taps, silu};
    return SEQ_TYPES(type, conv1d_step, a, (hipStream_t)stream);
}
