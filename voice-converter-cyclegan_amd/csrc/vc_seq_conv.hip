// vc_seq_conv.hip -- short causal convolution along the rows, one filter per channel: prompts, gradient, single frames.
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k];  y = p sigmoid(p) or p
//   g = dy * (p sigmoid(p))';  dx[u] = sum_k w[k] g[u + (K-1) - k];  dw[k] = sum_t g[t] x[t - (K-1) + k];  dbias = sum_t g[t]
// Bound by HBM.  A thread walks a run of rows for one 16-byte vector of channels with the last K frames in registers, so a row is fetched once,
// apart from the K - 1 frames ahead of a run.  Measured: 9001 x 1000 fp32 forward 17 us (4.3 TB/s of a copy's 5.0), 8192 x 2048 bf16 15.4 us, 4.4 TB/s.
#include "vc_seq.h"

struct ConvArgs { vc_conv1d_args a; SeqMap m; int v, cv, cvb, run, runs; bool past; float* part; };   // v channels a thread, cv such vectors, cvb of them next to each other; runs of `run` rows

// the utterance row r >= seq_head lies in: the last s with begin(s) <= r; n_seqs where r lies behind the last utterance
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
// Longest and shortest run of rows, and the waves below which a run is halved (a quarter of them once it has four rows).  Long runs repeat fewer frames ahead of them (the gradient: and behind
// them, with their sigmoids), short ones leave enough threads.  (Before stores went past the L2s.)  Gradient of 8192 x 2048 bf16, 4 taps, with its forward pass: 45.7 us by runs of 32, 51.7
// by 16, 55.8 by 64; of 1024 x 512: 14.4 by 4, 15.1 by 2, 15.6 by 8, 23.7 by 32; of 92 x 37 in 60 utterances: 24 by 2, 39 by 8.  Forward alone, 9001 x 1000 fp32: 17.2 by 8, 17.7 by 4 and by 16.
constexpr int FWD_RUN = 8, BWD_RUN = 32, SHORT_RUN = 2, RUN_WAVES = 1024;
// Rows worked on while as many are on their way: with two in the forward pass 18.0 us in place of 17.2, in the gradient 48.9 in place of 45.7.
constexpr int AHEAD = 4;
constexpr int BWD_V = 4;                                         // channels of a thread of the gradient
constexpr int FWD_WIDE = 32, BWD_WIDE = 64;                      // most vectors of channels next to each other in a block
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
struct Place { int c, run, base; bool ok; };                     // base: first row of the block's first run
__device__ __forceinline__ Place place(const ConvArgs& k, int V) {
    const int blocks = (k.cv + k.cvb - 1) / k.cvb;
    Place p;
    const int v = (int)(blockIdx.x % blocks) * k.cvb + threadIdx.x % k.cvb;
    const int first = (int)(blockIdx.x / blocks) * (256 / k.cvb);
    p.run = first + threadIdx.x / k.cvb;
    p.base = min(first, k.runs - 1) * k.run;
    // the last vector ends with the last channel: where V does not divide the channels it works out some of its neighbour's once more, to the same
    // values, and no access has to ask how many channels are left (fewer than V of them: V = 1)
    p.c = min(v * V, k.a.cols - V); p.ok = v < k.cv;
    return p;
}

// The rows that a block's threads work on, of one tensor, through a buffer descriptor: a row is a 32-bit offset (one addition from row to row), rows behind
// the tensor read as zeros, and an offset of NOWHERE reads zeros and stores nothing, which serves in place of branches.  Host code sees to it that a
// block's rows span less than 2^31 bytes.
constexpr unsigned NOWHERE = 0xf0000000u;
template <class T, int V> struct Span {
    __amdgpu_buffer_rsrc_t rs; unsigned ld;                      // bytes from row to row
    __device__ __forceinline__ Span(const void* p, int64_t stride, int base, int rows, int cols) : ld((unsigned)stride * (unsigned)sizeof(T)) {
        const int64_t bytes = ((int64_t)(rows - base - 1) * stride + cols) * (int64_t)sizeof(T);
        rs = __builtin_amdgcn_make_buffer_rsrc((void*)((const T*)p + (int64_t)base * stride), 0, (int)min(bytes, (int64_t)0x7fffffff), 0x00020000);
    }
    // PAST: the L2s are not to keep it
    template <bool PAST> __device__ __forceinline__ void store(unsigned at, const float (&f)[V]) const {
        constexpr int POLICY = PAST ? 2 : 0;                     // non-temporal or not
        Pack<T, V> q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = (T)f[i];
        if constexpr (V * sizeof(T) == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, q), rs, at, 0, POLICY);
        else if constexpr (V * sizeof(T) == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, q), rs, at, 0, POLICY);
        else if constexpr (V * sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, q), rs, at, 0, POLICY);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, q), rs, at, 0, POLICY);
    }
};
// V elements as they came: 16-bit ones two to a register
template <class T, int V> struct Raw {
    static constexpr int N = (V * (int)sizeof(T) + 3) / 4;
    unsigned w[N];
    __device__ __forceinline__ void load(const Span<T, V>& s, unsigned at) {
        if constexpr (N == 4) { const u32x4 q = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(s.rs, at, 0, 0)); w[0] = q[0]; w[1] = q[1]; w[2] = q[2]; w[3] = q[3]; }
        else if constexpr (N == 2) { const u32x2 q = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(s.rs, at, 0, 0)); w[0] = q[0]; w[1] = q[1]; }
        else if constexpr (sizeof(T) == 4) w[0] = __builtin_amdgcn_raw_buffer_load_b32(s.rs, at, 0, 0);
        else w[0] = __builtin_amdgcn_raw_buffer_load_b16(s.rs, at, 0, 0);
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (sizeof(T) == 4) f[i] = __builtin_bit_cast(float, w[i]);
            else f[i] = (float)__builtin_bit_cast(T, (unsigned short)(w[i / 2] >> (16 * (i % 2))));
        }
    }
};
template <class T, int K, int V, bool SILU, bool PAST> __global__ __launch_bounds__(256) void conv1d_fwd_kernel(const ConvArgs k) {
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
    int r = p.run * k.run;
    const int r1 = min(r + k.run, k.m.rows);
    const Span<T, V> X(a.x, a.x_ld, p.base, k.m.rows, a.cols), Y(a.y, a.y_ld, p.base, k.m.rows, a.cols);
    const unsigned ch = p.c * (unsigned)sizeof(T);
    for (const int head = min(seq_head(k.m), r1); r < head; ++r) {           // rows ahead of the first utterance
        const float f[V] = {};
        if (a.zero_tail) Y.template store<PAST>((r - p.base) * Y.ld + ch, f);
    }
    for (int s = seq_of(k.m, r); r < r1; ++s) {
        if (s >= k.m.n_seqs) {                                   // rows behind the last utterance
            const float f[V] = {};
            if (a.zero_tail) for (; r < r1; ++r) Y.template store<PAST>((r - p.base) * Y.ld + ch, f);
            return;
        }
        const int b = seq_begin(k.m, s), hi = min(seq_end(k.m, s, b), r1);
        if (r >= hi) continue;                                   // an empty utterance
        float win[K][V];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) frame<T, V>(a, s, b, r - b - (K - 1) + i, p.c, win[i]);
        unsigned from = (r - p.base) * X.ld + ch, to = (r - p.base) * Y.ld + ch;
        // AHEAD rows are worked on while the next are on their way; what rows past the end give is dropped
        Raw<T, V> next[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) next[i].load(X, from + i * X.ld);
        for (; r < hi; r += AHEAD) {
            Raw<T, V> now[AHEAD];
            from += AHEAD * X.ld;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) { now[i] = next[i]; next[i].load(X, r + AHEAD < hi ? from + i * X.ld : NOWHERE); }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                now[i].get(win[K - 1]);
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float q = w.b[e];
#pragma unroll
                    for (int j = 0; j < K; ++j) q = fmaf(w.w[j][e], win[j][e], q);
                    o[e] = SILU ? q * sigmoid<T>(q) : q;
#pragma unroll
                    for (int j = 0; j < K - 1; ++j) win[j][e] = win[j + 1][e];
                }
                Y.template store<PAST>(r + i < hi ? to + i * Y.ld : NOWHERE, o);
            }
            to += AHEAD * Y.ld;
        }
        r = hi;
    }
}

// g of one frame, from the K frames it looks at
template <class T, bool SILU, int K, int V> __device__ __forceinline__ void pre_gradient(const float (&win)[K][V], const float (&w)[K][V], const float (&b)[V], float (&g)[V]) {
    if constexpr (!SILU) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float q = b[e];
#pragma unroll
        for (int i = 0; i < K; ++i) q = fmaf(w[i][e], win[i][e], q);
        const float sg = sigmoid<T>(q);
        g[e] *= sg * fmaf(q, 1.f - sg, 1.f);
    }
}
// A run's dx needs the K - 1 frames' g behind it as well: they are worked out again there.  dx of a frame gathers in a register ring while the
// frames that look at it go by.
// 8192 x 2048 bf16: 23 to 25 us, 4.2 TB/s, the vector units busy 82 % of the time with the pre-activation and its sigmoid once more.
// Four channels a thread: eight would fill the registers (filter, window, ring and its share of dw are K vectors each) and leave too few waves to wait with.
template <class T, int K, int V, bool SILU, bool PAST> __global__ __launch_bounds__(256) void conv1d_bwd_kernel(const ConvArgs k) {
    __shared__ float red[256 * V];
    const vc_conv1d_args& a = k.a;
    const Place p = place(k, V);
    float dw[K][V] = {}, db[V] = {};
    if (p.ok && p.run < k.runs) {
        const Filter<T, K, V> w(a, p.c);
        int r = p.run * k.run;
        const int r1 = min(r + k.run, k.m.rows);
        const bool want_dx = a.dx != nullptr;
        const Span<T, V> X(a.x, a.x_ld, p.base, k.m.rows, a.cols), DY(a.dy, a.dy_ld, p.base, k.m.rows, a.cols),
            DX(want_dx ? a.dx : a.dy, want_dx ? a.dx_ld : a.dy_ld, p.base, k.m.rows, a.cols);
        const unsigned ch = p.c * (unsigned)sizeof(T);
        for (const int head = min(seq_head(k.m), r1); r < head; ++r) {
            const float f[V] = {};
            if (a.zero_tail && want_dx) DX.template store<PAST>((r - p.base) * DX.ld + ch, f);
        }
        for (int s = seq_of(k.m, r); r < r1; ++s) {
            if (s >= k.m.n_seqs) {
                const float f[V] = {};
                if (a.zero_tail && want_dx) for (; r < r1; ++r) DX.template store<PAST>((r - p.base) * DX.ld + ch, f);
                break;
            }
            const int b = seq_begin(k.m, s), end = seq_end(k.m, s, b), lo = r, hi = min(end, r1);
            if (lo >= hi) continue;
            float win[K][V], ring[K][V] = {};                    // ring[i]: dx of frame r - (K-1) + i so far
#pragma unroll
            for (int i = 0; i < K - 1; ++i) frame<T, V>(a, s, b, lo - b - (K - 1) + i, p.c, win[i]);
            // K - 1 rows more than the run's: their g where the utterance has them, zeros behind its end.  AHEAD rows are worked on while the next are
            // on their way
            const int stop = want_dx ? hi + K - 1 : hi;
            unsigned xo = (r - p.base) * X.ld + ch, go = (r - p.base) * DY.ld + ch, to = (r - (K - 1) - p.base) * DX.ld + ch;
            Raw<T, V> xn[AHEAD], gn[AHEAD];
            auto fetch = [&](int at) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const bool in = at + i < min(end, stop);
                    xn[i].load(X, in ? xo + i * X.ld : NOWHERE); gn[i].load(DY, in ? go + i * DY.ld : NOWHERE);
                }
                xo += AHEAD * X.ld; go += AHEAD * DY.ld;
            };
            fetch(r);
            for (; r < stop; r += AHEAD) {
                Raw<T, V> xc[AHEAD], gc[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) { xc[i] = xn[i]; gc[i] = gn[i]; }
                fetch(r + AHEAD);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    float g[V];
                    xc[i].get(win[K - 1]); gc[i].get(g);
                    pre_gradient<T, SILU, K, V>(win, w.w, w.b, g);
                    const bool mine = r + i < hi;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float gm = mine ? g[e] : 0.f;
                        db[e] += gm;
#pragma unroll
                        for (int j = 0; j < K; ++j) {
                            dw[j][e] = fmaf(gm, win[j][e], dw[j][e]);
                            ring[j][e] = j == K - 1 ? w.w[j][e] * g[e] : fmaf(w.w[j][e], g[e], ring[j][e]);
                        }
                    }
                    const int at = r + i - (K - 1);              // has all its shares now, but that of the final state's gradient
                    if (a.dfinal && at >= lo && at < hi && at >= end - (K - 1)) {
                        float o[V];
                        load_vec<T, V>((const T*)a.dfinal + ((int64_t)s * (K - 1) + at - (end - (K - 1))) * a.cols + p.c, o);
#pragma unroll
                        for (int e = 0; e < V; ++e) ring[0][e] += o[e];
                    }
                    DX.template store<PAST>(want_dx && at >= lo && at < hi ? to + i * DX.ld : NOWHERE, ring[0]);
#pragma unroll
                    for (int e = 0; e < V; ++e)
#pragma unroll
                        for (int j = 0; j < K - 1; ++j) { win[j][e] = win[j + 1][e]; ring[j][e] = ring[j + 1][e]; }
                }
                to += AHEAD * DX.ld;
            }
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
            pre_gradient<T, SILU, K, V>(win, w.w, w.b, g);
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
// One frame: a channel a thread, no more than latency.  8 streams x 1024: 3.0 us, of which an empty launch is 2.
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
    *y = (T)(a.silu ? p * sigmoid<T>(p) : p);
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
    VC_ARG(a->rows >= 0 && a->rows + (int64_t)std::max(a->n_seqs, 0) < (1LL << 31) - (1 << 16) && a->cols > 0 && a->cols <= SEQ_COLS && a->n_seqs > 0, "%s: bad sizes (rows %lld, cols %d, n_seqs %d)", who, (long long)a->rows, a->cols, a->n_seqs);
    VC_ARG(a->offsets || a->rows % a->n_seqs == 0, "%s: without offsets the rows divide into n_seqs equal utterances", who);
    k->a = *a;
    k->m = SeqMap{a->offsets, (int)a->rows, a->n_seqs, (int)(a->rows / a->n_seqs)};
    k->v = a->cols < v ? 1 : v;
    k->cv = (a->cols + k->v - 1) / k->v;
    for (k->cvb = 1; k->cvb < k->cv && k->cvb < most;) k->cvb *= 2;
    k->part = nullptr;
    k->past = a->rows * a->cols * seq_esize(a->type) >= STREAM_BYTES;
    return 0;
}
static void set_runs(ConvArgs& k, int longest) {
    for (k.run = longest; k.run > SHORT_RUN && (int64_t)k.m.rows * k.cv < (int64_t)k.run * 64 * (k.run > 4 ? RUN_WAVES : RUN_WAVES / 4);) k.run /= 2;
    k.runs = (k.m.rows + k.run - 1) / k.run;
}
static int conv_grid(const char* who, const ConvArgs& k, bool seqs, int64_t out_ld, unsigned* grid) {
    const int per = 256 / k.cvb;
    const int64_t g = (int64_t)((k.cv + k.cvb - 1) / k.cvb) * (((int64_t)k.runs + (seqs ? k.m.n_seqs : 0) + per - 1) / per);
    VC_ARG(g < (1LL << 31), "%s: too many rows and channels for one launch", who);
    // the rows of a block, with the frames that its runs look at ahead and behind, by 32-bit offsets
    const int64_t span = std::min((int64_t)per * k.run, (int64_t)k.m.rows) + 16;
    for (int64_t ld : {k.a.x_ld, k.a.y ? k.a.y_ld : 0, k.a.dy ? k.a.dy_ld : 0, k.a.dx ? k.a.dx_ld : 0})
        VC_ARG(ld >= 0 && (span * ld + k.a.cols) * seq_esize(k.a.type) < (1LL << 31), "%s: a row stride of %lld elements is out of range", who, (long long)ld);
    VC_ARG(k.m.rows <= 1 || out_ld >= k.a.cols, "%s: a row stride of %lld elements: rows of an output of %d channels overlap", who, (long long)out_ld, k.a.cols);
    *grid = (unsigned)g;
    return 0;
}
template <class T, int K> static int fwd_k(const ConvArgs& k, unsigned grid, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
#define F(V, SILU, PAST) hipLaunchKernelGGL((conv1d_fwd_kernel<T, K, V, SILU, PAST>), dim3(grid), dim3(256), 0, s, k)
    if (k.v == 1) { if (k.a.silu) F(1, true, false); else F(1, false, false); }       // fewer channels than a vector
    else if (k.past) { if (k.a.silu) F(V, true, true); else F(V, false, true); }
    else if (k.a.silu) F(V, true, false);
    else F(V, false, false);
#undef F
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T, int K> static int bwd_k(const ConvArgs& k, unsigned grid, hipStream_t s) {
    constexpr int V = BWD_V;
#define F(V, SILU, PAST) hipLaunchKernelGGL((conv1d_bwd_kernel<T, K, V, SILU, PAST>), dim3(grid), dim3(256), 0, s, k)
    if (k.v == 1) { if (k.a.silu) F(1, true, false); else F(1, false, false); }       // fewer channels than a vector
    else if (k.past) { if (k.a.silu) F(V, true, true); else F(V, false, true); }
    else if (k.a.silu) F(V, true, false);
    else F(V, false, false);
#undef F
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
    set_runs(k, FWD_RUN);
    unsigned grid; VC_CHECK(conv_grid("vc_causal_conv1d_fwd", k, a->final_state != nullptr, a->y_ld, &grid));
    VC_ARG(a->rows == 0 || a->y != a->x, "vc_causal_conv1d_fwd: not in place: a run of rows looks at frames that another one writes");
    return SEQ_TYPES(a->type, conv1d_fwd, k, grid, (hipStream_t)stream);
}
// rows of `part`: one for each block's runs
static int conv_parts(const ConvArgs& k) { const int per = 256 / k.cvb; return (k.runs + per - 1) / per; }
extern "C" int64_t vc_causal_conv1d_bwd_work(const vc_conv1d_args* a) {
    ConvArgs k; if (check_conv1d("vc_causal_conv1d_bwd_work", a, BWD_V, BWD_WIDE, &k)) return VC_E_ARG;
    set_runs(k, BWD_RUN);
    return (int64_t)conv_parts(k) * (a->taps + 1) * a->cols;
}
extern "C" int vc_causal_conv1d_bwd(const vc_conv1d_args* a, void* stream) {
    ConvArgs k; VC_CHECK(check_conv1d("vc_causal_conv1d_bwd", a, BWD_V, BWD_WIDE, &k));
    VC_ARG(a->w && (a->rows == 0 || (a->x && a->dy)), "vc_causal_conv1d_bwd: null pointer");
    set_runs(k, BWD_RUN);
    const bool params = a->dw || a->dbias;
    const int64_t need = (int64_t)conv_parts(k) * (a->taps + 1) * a->cols;
    if (params && need && (!a->work || a->work_floats < need)) { vc_set_error("vc_causal_conv1d_bwd: work is too small (%lld floats needed)", (long long)need); return VC_E_NOMEM; }
    if (params) k.part = a->work;
    unsigned grid; VC_CHECK(conv_grid("vc_causal_conv1d_bwd", k, a->dinitial != nullptr, a->dx ? a->dx_ld : a->cols, &grid));
    VC_ARG((!a->dx || a->rows == 0 || (a->dx != a->x && a->dx != a->dy)) && (!a->dinitial || (a->dinitial != a->initial && a->dinitial != a->dfinal)),
           "vc_causal_conv1d_bwd: not in place: a run of rows looks at frames that another one writes");
    if (grid) VC_CHECK(SEQ_TYPES(a->type, conv1d_bwd, k, grid, (hipStream_t)stream));
    // no rows: no parts, and the sums are zeros
    return params ? seq_sum_parts(k.part, conv_parts(k), (int64_t)(a->taps + 1) * a->cols, a->dw, (int64_t)a->taps * a->cols, a->dbias, (hipStream_t)stream) : 0;
}
extern "C" int vc_causal_conv1d_step(const void* x, int64_t x_ld, void* state, const int32_t* slots, const float* w, const float* bias,
                                     void* y, int64_t y_ld, int rows, int n_slots, int cols, int taps, int type, int silu, void* stream) {
    VC_ARG(seq_type_ok(type), "vc_causal_conv1d_step: type must be VC_F32, VC_BF16 or VC_F16");
    VC_ARG(taps >= 2 && taps <= 8, "vc_causal_conv1d_step: 2 to 8 taps, got %d", taps);
    VC_ARG(rows >= 0 && rows <= 65535 && n_slots > 0 && cols > 0 && cols <= SEQ_COLS, "vc_causal_conv1d_step: bad sizes (rows %d, n_slots %d, cols %d)", rows, n_slots, cols);
    VC_ARG(slots || rows <= n_slots, "vc_causal_conv1d_step: %d rows without slots, and %d slots", rows, n_slots);
    VC_ARG(!slots || rows <= MAX_SLOT_ROWS, "vc_causal_conv1d_step: at most %d rows with slots, got %d", MAX_SLOT_ROWS, rows);
    if (rows == 0) return 0;
    VC_ARG(x && state && w && y, "vc_causal_conv1d_step: null pointer");
    VC_ARG(rows == 1 || (x_ld >= 0 && y_ld >= cols), "vc_causal_conv1d_step: a row stride is out of range, or rows of y overlap");
    const ConvStepArgs a{x, state, slots, w, bias, y, x_ld, y_ld, rows, n_slots, cols, taps, silu};
    return SEQ_TYPES(type, conv1d_step, a, (hipStream_t)stream);
}
