// vc_seq_norm.hip -- RMS norm of a frame's channels with the residual's addition, its 8-bit form, its gradient.
//   t = x + residual (as stored);  y = t * rstd * gamma,  rstd = 1 / sqrt(mean(t^2) + eps)
//   dt = dsum + rstd * (g - that * mean(g * that)),  g = dy * gamma, that = t * rstd;   dgamma = sum over rows of dy * that
// All of it is bound by HBM: a row is read once into registers (TPR threads hold it, ITEMS 16-byte vectors each), its sum taken there, and written.
#include "vc_seq.h"

struct NormRowArgs {
    const void* x; const void* res; const float* gamma; void* y; void* sum; float* rstd; float* scale;
    const void* dy; const void* dsum; void* dx; void* dres; float* part;
    int64_t x_ld, res_ld, y_ld, sum_ld, dy_ld, dsum_ld, dx_ld, dres_ld;
    float eps; int64_t rows; int cols, group; bool past, past_in;     // stores, loads that go past the L2s
};

// sum / largest over the TPR threads of a row; every one gets it.  TPR = 64: a wave, no barrier; else the block
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum_dpp(v);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}
template <int LANES> __device__ __forceinline__ unsigned lanes_max(unsigned v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}
template <int TPR> __device__ __forceinline__ unsigned row_max(unsigned v, float* red) {
    v = lanes_max<64>(v);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __uint_as_float(v);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v = max(v, __float_as_uint(red[i]));
    }
    return v;
}
template <int TPR> __device__ __forceinline__ float row_maxf(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v = fmaxf(v, red[i]);
    }
    return v;
}
// four (V = 4) or eight values as e4m3: rounded to nearest even by the conversion instruction; |f| <= 448 (1 + 2^-23), which rounds to 448
template <int V> __device__ __forceinline__ void store_e4m3(unsigned char* p, const float (&f)[V], int n) {
    unsigned w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
        w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], lo, true);
    }
    if (n >= V) {
        struct __attribute__((packed, aligned(1))) W { unsigned v[V / 4]; } q;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) q.v[i] = w[i];
        *(W*)p = q;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < n) p[i] = (unsigned char)(w[i / 4] >> (8 * (i % 4)));
    }
}
// The largest |t gamma| of a group as an integer: ordered like the numbers, a NaN above infinity (fmaxf would drop it)
constexpr float E4M3_TOP = 448.f, LEAST_TOP = 0x1p-100f;
template <int V> __device__ __forceinline__ unsigned top_of(const float (&f)[V], unsigned m) {
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(fabsf(f[i])));
    return m;
}
// y / scale of a group.  rstd falls out of it: q = t gamma * 448 / max|t gamma|.  A quotient next to a border between two of the 8-bit values goes to the
// wrong one where its fp32 error reaches across (a few in a million elements), so what the products and the division round off is carried along: e is
// the rounding error of t gamma (rest: that of the largest), one multiply-add each.  A group under the least scale (rows of zeros, above all) takes that.
// Their sum is rounded to odd: fp32 holds every border, and a sum that is not exact must not become one (to nearest, a quotient within 2^-25 of a border
// would, and the tie would send it to the even side).  What is left out is 2^-45 of the value: none of 17 million values on the wrong side.
struct Quant { float first, factor, correction, scale; };
__device__ __forceinline__ Quant quant_of(unsigned bits, float rest, float rstd) {
    const float top = __uint_as_float(bits), y = top * rstd;
    Quant q;
    if (y >= LEAST_TOP) {                                        // (448 / top would leave fp32 below 2^-119: products that small take 2^100 first)
        q.first = top < 0x1p-100f ? 0x1p100f : 1.f;
        const float t = top * q.first;
        q.factor = E4M3_TOP / t; q.scale = y / E4M3_TOP;
        q.correction = (fmaf(-q.factor, t, E4M3_TOP) - q.factor * (rest * q.first)) / E4M3_TOP;
    } else { q.first = rstd; q.factor = E4M3_TOP / LEAST_TOP; q.correction = 0.f; q.scale = y != y ? y : LEAST_TOP / E4M3_TOP; }
    return q;
}
__device__ __forceinline__ float quantised(const Quant& k, float p, float e) {
#pragma clang fp contract(off)                                    // q is the rounded product: folded into q + r its error would count twice
    const float v = p * k.first, q = v * k.factor, r = fmaf(v, k.factor, -q) + fmaf(e * k.first, k.factor, q * k.correction), s = q + r, rest = r - (s - q);
    const int bits = __float_as_int(s);                          // the sum is off by `rest`: one step that way where its last bit is even
    return __int_as_float(rest == 0.f || (bits & 1) ? bits : bits + ((rest < 0.f) == (bits < 0) ? 1 : -1));
}
// the rounding error of the largest |t gamma|: of several, the one that makes it largest
template <int V> __device__ __forceinline__ float rest_of(const float (&p)[V], const float (&e)[V], unsigned top, float m) {
#pragma unroll
    for (int i = 0; i < V; ++i) m = __float_as_uint(fabsf(p[i])) == top ? fmaxf(m, copysignf(1.f, p[i]) * e[i]) : m;
    return m;
}
constexpr float NO_REST = -3.0e38f;

// A row of up to TPR * ITEMS vectors in registers.  Threads walk the rows with a stride of the grid, so gamma is read once for all of them.
// 16384 x 1024 bf16 with a residual: 28 us, 4.8 TB/s (a copy 5.0); 8832 x 2048 bf16 on an fp32 stream to 8 bits: 39 us, 5.1 TB/s; 1 x 512: 2.9 us.
template <class T, class S, bool E4M3, int TPR, int ITEMS> __global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_fwd_kernel(const NormRowArgs a) {
    constexpr int V = 16 / (int)sizeof(T), RPB = TPR == 64 ? 4 : 1;
    __shared__ float red[TPR / 64 > 0 ? TPR / 64 : 1];
    const int t = threadIdx.x % TPR;
    float gm[ITEMS][V];
    int left[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int c = (i * TPR + t) * V;
        left[i] = a.cols - c;
#pragma unroll
        for (int e = 0; e < V; ++e) gm[i][e] = 0.f;
        if (left[i] > 0) load_some<float, V>(a.gamma + c, gm[i], left[i]);
    }
    const float inv_cols = 1.f / (float)a.cols;
    for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < a.rows; r += (int64_t)gridDim.x * RPB) {
        float f[ITEMS][V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = (i * TPR + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) f[i][e] = 0.f;
            if (left[i] > 0) load_in<T, V>((const T*)a.x + r * a.x_ld + c, f[i], left[i], a.past_in);
        }
        if (a.res) {
            float g[ITEMS][V];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = (i * TPR + t) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) g[i][e] = 0.f;
                if (left[i] > 0) load_in<S, V>((const S*)a.res + r * a.res_ld + c, g[i], left[i], a.past_in);
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = (i * TPR + t) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) f[i][e] = (float)(S)(f[i][e] + g[i][e]);
                if (left[i] > 0) store_out<S, V>((S*)a.sum + r * a.sum_ld + c, f[i], left[i], a.past);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(f[i][e], f[i][e], ss);
        const float rstd = 1.f / sqrtf(row_sum<TPR>(ss, red) * inv_cols + a.eps);
        if (a.rstd && t == 0) a.rstd[r] = rstd;
        float err[E4M3 ? ITEMS : 1][V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (E4M3) { const float p = f[i][e] * gm[i][e]; err[i][e] = fmaf(f[i][e], gm[i][e], -p); f[i][e] = p; }
                else f[i][e] = f[i][e] * rstd * gm[i][e];
            }
        if constexpr (!E4M3) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (left[i] > 0) store_out<T, V>((T*)a.y + r * a.y_ld + (i * TPR + t) * V, f[i], left[i], a.past);
        } else {
            Quant k[ITEMS];
            if (a.group == 0) {
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) m = top_of<V>(f[i], m);
                m = row_max<TPR>(m, red);
                float rest = NO_REST;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) rest = rest_of<V>(f[i], err[i], m, rest);
                k[0] = quant_of(m, row_maxf<TPR>(rest, red), rstd);
                if (t == 0) a.scale[r] = k[0].scale;
#pragma unroll
                for (int i = 1; i < ITEMS; ++i) k[i] = k[0];
            } else {
                const int gl = a.group / V;                      // lanes that share a scale: 4 to 32, next to each other
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    unsigned m = top_of<V>(f[i], 0);
                    for (int o = 1; o < gl; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
                    float rest = rest_of<V>(f[i], err[i], m, NO_REST);
                    for (int o = 1; o < gl; o <<= 1) rest = fmaxf(rest, __shfl_xor(rest, o, 64));
                    k[i] = quant_of(m, rest, rstd);
                    if (left[i] > 0 && t % gl == 0) a.scale[r * (a.cols / a.group) + (i * TPR + t) / gl] = k[i].scale;
                }
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float q[V];
#pragma unroll
                for (int e = 0; e < V; ++e) q[e] = quantised(k[i], f[i][e], err[i][e]);
                if (left[i] > 0) store_e4m3<V>((unsigned char*)a.y + r * a.y_ld + (i * TPR + t) * V, q, left[i]);
            }
        }
    }
}
// Rows longer than the registers of a block hold: one block a row, which it reads again for each pass (out of L2)
template <class T, class S, bool E4M3> __global__ __launch_bounds__(1024) void rms_fwd_long_kernel(const NormRowArgs a) {
    __shared__ float red[16];
    const int64_t r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.x_ld;
    const S* res = a.res ? (const S*)a.res + r * a.res_ld : nullptr;
    S* sum = a.res ? (S*)a.sum + r * a.sum_ld : nullptr;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
        float f = (float)x[c];
        if (res) { const S q = (S)(f + (float)res[c]); sum[c] = q; f = (float)q; }
        ss = fmaf(f, f, ss);
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(ss, red) / (float)a.cols + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    auto t = [&](int c) { return sum ? (float)sum[c] : (float)x[c]; };                            // a thread reads back what it wrote itself
    if constexpr (!E4M3) {
        for (int c = threadIdx.x; c < a.cols; c += 1024) ((T*)a.y)[r * a.y_ld + c] = (T)(t(c) * rstd * a.gamma[c]);
    } else {
        // scales: a wave for each group of 64 threads' columns would leave most idle, so each pass of the block covers 1024 columns: 8 to 32 groups
        auto product = [&](int c, float& e) { const float f = t(c), g = a.gamma[c], p = f * g; e = fmaf(f, g, -p); return p; };
        Quant k{};
        if (a.group == 0) {
            unsigned m = 0;
            float e, rest = NO_REST;
            for (int c = threadIdx.x; c < a.cols; c += 1024) m = max(m, __float_as_uint(fabsf(product(c, e))));
            m = row_max<1024>(m, red);
            for (int c = threadIdx.x; c < a.cols; c += 1024) { const float p[1] = {product(c, e)}, q[1] = {e}; rest = rest_of<1>(p, q, m, rest); }
            k = quant_of(m, row_maxf<1024>(rest, red), rstd);
            if (threadIdx.x == 0) a.scale[r] = k.scale;
        }
        __shared__ unsigned top[1024 / 32];
        __shared__ float most[1024 / 32];
        for (int c0 = 0; c0 < a.cols; c0 += 1024) {              // 1024 columns at a time: 8 to 32 groups
            const int c = c0 + threadIdx.x;
            float e = 0.f;
            const float p = c < a.cols ? product(c, e) : 0.f;
            if (a.group) {
                const int per = a.group / 32, first = threadIdx.x / a.group * per;
                unsigned m = lanes_max<32>(__float_as_uint(fabsf(p)));
                __syncthreads();
                if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
                __syncthreads();
                for (int i = 0; i < per; ++i) m = max(m, top[first + i]);
                const float p1[1] = {p}, e1[1] = {e};
                float rest = rest_of<1>(p1, e1, m, NO_REST);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) rest = fmaxf(rest, __shfl_xor(rest, o, 64));
                if (threadIdx.x % 32 == 0) most[threadIdx.x / 32] = rest;
                __syncthreads();
                for (int i = 0; i < per; ++i) rest = fmaxf(rest, most[first + i]);
                k = quant_of(m, rest, rstd);
                if (c < a.cols && threadIdx.x % a.group == 0) a.scale[r * (a.cols / a.group) + c / a.group] = k.scale;
            }
            const float q = quantised(k, p, e);
            if (c < a.cols) ((unsigned char*)a.y)[r * a.y_ld + c] = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
        }
    }
}

// Gradient.  Every thread keeps its columns' share of dgamma over all rows it walks; a block leaves one row of `part`.  16384 x 1024 bf16: 30 us, 4.4 TB/s.
template <class T, class S, int TPR, int ITEMS> __global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_bwd_kernel(const NormRowArgs a) {
    constexpr int V = 16 / (int)sizeof(T), RPB = TPR == 64 ? 4 : 1;
    __shared__ float red[TPR / 64 > 0 ? TPR / 64 : 1];
    const int t = threadIdx.x % TPR;
    float gm[ITEMS][V], dg[ITEMS][V];
    int left[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int c = (i * TPR + t) * V;
        left[i] = a.cols - c;
#pragma unroll
        for (int e = 0; e < V; ++e) { gm[i][e] = 0.f; dg[i][e] = 0.f; }
        if (left[i] > 0) load_some<float, V>(a.gamma + c, gm[i], left[i]);
    }
    const float inv_cols = 1.f / (float)a.cols;
    for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < a.rows; r += (int64_t)gridDim.x * RPB) {
        float th[ITEMS][V], g[ITEMS][V], ds[ITEMS][V];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = (i * TPR + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { th[i][e] = 0.f; g[i][e] = 0.f; ds[i][e] = 0.f; }
            if (left[i] > 0) {
                load_in<S, V>((const S*)a.sum + r * a.sum_ld + c, th[i], left[i], a.past_in);
                load_in<T, V>((const T*)a.dy + r * a.dy_ld + c, g[i], left[i], a.past_in);
                if (a.dsum) load_in<S, V>((const S*)a.dsum + r * a.dsum_ld + c, ds[i], left[i], a.past_in);
            }
        }
        const float rstd = a.rstd[r];
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                th[i][e] *= rstd;
                dg[i][e] = fmaf(g[i][e], th[i][e], dg[i][e]);
                g[i][e] *= gm[i][e];
                m = fmaf(g[i][e], th[i][e], m);
            }
        if (!a.dx && !a.dres) continue;                          // the same for all threads
        m = row_sum<TPR>(m, red) * inv_cols;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = (i * TPR + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) g[i][e] = fmaf(rstd, fmaf(-th[i][e], m, g[i][e]), ds[i][e]);
            if (left[i] <= 0) continue;
            if (a.dx) store_out<T, V>((T*)a.dx + r * a.dx_ld + c, g[i], left[i], a.past);
            if (a.dres) store_out<S, V>((S*)a.dres + r * a.dres_ld + c, g[i], left[i], a.past);
        }
    }
    if (!a.part) return;
    if constexpr (RPB > 1) {                                     // the block's rows of threads, one behind the other
        __shared__ float acc[TPR * ITEMS * V];
        for (int w = 0; w < RPB; ++w) {
            if ((int)threadIdx.x / TPR == w)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float& p = acc[(i * V + e) * TPR + t];
                        dg[i][e] += w ? p : 0.f;
                        p = dg[i][e];
                    }
            __syncthreads();
        }
        if ((int)threadIdx.x / TPR != RPB - 1) return;           // the last one holds the sums
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (left[i] > 0) store_some<float, V>(a.part + (int64_t)blockIdx.x * a.cols + (i * TPR + t) * V, dg[i], left[i]);
}
template <class T, class S> __global__ __launch_bounds__(1024) void rms_bwd_long_kernel(const NormRowArgs a) {
    __shared__ float red[16];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const S* t = (const S*)a.sum + r * a.sum_ld;
        const T* dy = (const T*)a.dy + r * a.dy_ld;
        const S* ds = a.dsum ? (const S*)a.dsum + r * a.dsum_ld : nullptr;
        const float rstd = a.rstd[r];
        float* part = a.part ? a.part + (int64_t)blockIdx.x * a.cols : nullptr;
        float m = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float th = (float)t[c] * rstd, d = (float)dy[c];
            m = fmaf(d * a.gamma[c], th, m);
            if (part) part[c] = (r == blockIdx.x ? 0.f : part[c]) + d * th;
        }
        m = row_sum<1024>(m, red) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float d = fmaf(rstd, (float)dy[c] * a.gamma[c] - (float)t[c] * rstd * m, ds ? (float)ds[c] : 0.f);
            if (a.dx) ((T*)a.dx)[r * a.dx_ld + c] = (T)d;
            if (a.dres) ((S*)a.dres)[r * a.dres_ld + c] = (S)d;
        }
    }
}

// C columns a block, 1024 / C threads a column
template <int C> __global__ __launch_bounds__(1024) void sum_parts_kernel(const float* part, int parts, int64_t n, float* dst0, int64_t n0, float* dst1) {
    constexpr int W = 1024 / C;
    __shared__ float red[W][C + 1];
    const int64_t c = (int64_t)blockIdx.x * C + threadIdx.x % C;
    const int w = threadIdx.x / C;
    float s = 0.f;
    if (c < n) {
        int p = w;
        for (; p + 3 * W < parts; p += 4 * W) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = part[(int64_t)(p + W * i) * n + c];
#pragma unroll
            for (int i = 0; i < 4; ++i) s += v[i];
        }
        for (; p < parts; p += W) s += part[(int64_t)p * n + c];
    }
    red[w][threadIdx.x % C] = s;
    __syncthreads();
    if (w || c >= n) return;
    s = 0.f;
#pragma unroll 16
    for (int i = 0; i < W; ++i) s += red[i][threadIdx.x];
    float* dst = c < n0 ? dst0 : dst1;
    if (dst) dst[c < n0 ? c : c - n0] = s;
}
int seq_sum_parts(const float* part, int parts, int64_t n, float* dst0, int64_t n0, float* dst1, hipStream_t s) {
    // few columns: narrow blocks, so that there are enough of them.  1024 x 1024 floats: 3.7 us by 16 columns, 6.7 by 64
    if (n <= 16384) hipLaunchKernelGGL(sum_parts_kernel<16>, dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, s, part, parts, n, dst0, n0, dst1);
    else hipLaunchKernelGGL(sum_parts_kernel<64>, dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, s, part, parts, n, dst0, n0, dst1);
    VC_HIP(hipGetLastError());
    return 0;
}

// How a row of nv vectors is held: by a wave with up to two vectors a thread, which needs no barrier; longer ones by a block of 256, 512, then of 1024.
// (Before loads and stores went past the L2s.)  Rows of 2048 bf16 with 8-bit output (8832 of them): 58 us by a wave with four vectors a thread, whose registers leave four waves a SIMD, 53 by 128
// threads, 45 by 256; rows of 1024: 32 us by a wave, 40 by 128 or 256 threads; 2535 rows of 4352 to 8 bits: 40 us by 256 threads, 36 by 512, 38 by 1024.
#define NORM_LAYOUT(nv, F) \
    ((nv) <= 64 ? F(64, 1) : (nv) <= 128 ? F(64, 2) : (nv) <= 256 ? F(256, 1) : (nv) <= 512 ? F(256, 2) : (nv) <= 1024 ? F(512, 2) : F(1024, 2))
static int norm_tpr(int64_t nv) {                                // threads of a row: 64 (four rows a block), or a block
#define F(TPR, ITEMS) TPR
    return NORM_LAYOUT(nv, F);
#undef F
}
constexpr int64_t NORM_MOST = 2048;                              // vectors of the longest row that registers hold
static int64_t norm_vectors(int cols, int type) { const int v = 16 / seq_esize(type); return (cols + v - 1) / v; }

template <class T, class S, bool E, int TPR, int ITEMS> static void launch_fwd(const NormRowArgs& a, hipStream_t s) {
    const int64_t rpb = TPR == 64 ? 4 : 1, want = (a.rows + rpb - 1) / rpb;
    const int64_t most = TPR == 1024 ? 1024 : 4096;
    hipLaunchKernelGGL((rms_fwd_kernel<T, S, E, TPR, ITEMS>), dim3((unsigned)std::min(want, most)), dim3(TPR == 64 ? 256 : TPR), 0, s, a);
}
template <class T, class S, bool E> static int norm_fwd_e(const NormRowArgs& a, hipStream_t s) {
    const int64_t nv = (a.cols + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T));
    if (nv > NORM_MOST) hipLaunchKernelGGL((rms_fwd_long_kernel<T, S, E>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
    else {
#define F(TPR, ITEMS) launch_fwd<T, S, E, TPR, ITEMS>(a, s)
        NORM_LAYOUT(nv, F);
#undef F
    }
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int norm_fwd(const NormRowArgs& a, bool wide, bool e4m3, hipStream_t s) {
    if (wide) return e4m3 ? norm_fwd_e<T, float, true>(a, s) : norm_fwd_e<T, float, false>(a, s);
    return e4m3 ? norm_fwd_e<T, T, true>(a, s) : norm_fwd_e<T, T, false>(a, s);
}
// Blocks of the gradient: enough to fill the card, few enough that their rows of `part` cost little beside the activations
static int norm_bwd_blocks(int64_t rows, int cols, int type) {
    const int tpr = norm_tpr(norm_vectors(cols, type));
    const int64_t rpb = tpr == 64 ? 4 : 1, most = tpr == 1024 ? 256 : 1024;
    return (int)std::min<int64_t>((rows + rpb - 1) / rpb, most);
}
template <class T, class S, int TPR, int ITEMS> static void launch_bwd(const NormRowArgs& a, int blocks, hipStream_t s) {
    hipLaunchKernelGGL((rms_bwd_kernel<T, S, TPR, ITEMS>), dim3(blocks), dim3(TPR == 64 ? 256 : TPR), 0, s, a);
}
template <class T, class S> static int norm_bwd_t(const NormRowArgs& a, int type, float* dgamma, hipStream_t s) {
    const int64_t nv = norm_vectors(a.cols, type);
    const int blocks = norm_bwd_blocks(a.rows, a.cols, type);
    if (nv > NORM_MOST) hipLaunchKernelGGL((rms_bwd_long_kernel<T, S>), dim3(blocks), dim3(1024), 0, s, a);
    else {
#define F(TPR, ITEMS) launch_bwd<T, S, TPR, ITEMS>(a, blocks, s)
        NORM_LAYOUT(nv, F);
#undef F
    }
    VC_HIP(hipGetLastError());
    return dgamma ? seq_sum_parts(a.part, blocks, a.cols, dgamma, a.cols, nullptr, s) : 0;
}
template <class T> static int norm_bwd(const NormRowArgs& a, bool wide, int type, float* dgamma, hipStream_t s) {
    return wide ? norm_bwd_t<T, float>(a, type, dgamma, s) : norm_bwd_t<T, T>(a, type, dgamma, s);
}

static int check_norm(const char* who, int64_t rows, int cols, int type, int sum_type) {
    VC_ARG(rows >= 0 && rows < (1LL << 31) && cols > 0 && cols <= NORM_COLS, "%s: bad sizes (rows %lld, cols %d)", who, (long long)rows, cols);
    VC_ARG(seq_type_ok(type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(sum_type == type || sum_type == VC_F32, "%s: the residual stream has the activations' type or fp32", who);
    return 0;
}
// rows of an output closer than their width would be written by several threads in no order; a single row has no stride
static int check_ld(const char* who, const NormRowArgs& a, std::initializer_list<int64_t> in, std::initializer_list<int64_t> out) {
    if (a.rows <= 1) return 0;
    for (int64_t ld : in) VC_ARG(ld >= 0, "%s: a row stride of %lld elements is out of range", who, (long long)ld);
    for (int64_t ld : out) VC_ARG(ld >= a.cols, "%s: a row stride of %lld elements: rows of an output of %d columns overlap", who, (long long)ld, a.cols);
    return 0;
}
static void set_past(NormRowArgs& a, int type, bool wide) {
    const int64_t e = seq_esize(type), es = wide ? 4 : e, n = a.rows * a.cols;
    a.past = n * e >= STREAM_BYTES;
    const int64_t read = a.dy ? n * (e + (a.dsum ? 2 : 1) * es) : n * (e + (a.res ? es : 0));
    a.past_in = read >= LOAD_BYTES;
    for (int64_t w : {(int64_t)a.cols, a.x_ld, a.res_ld, a.sum_ld, a.dy_ld, a.dsum_ld}) a.past_in = a.past_in && w * e % 128 == 0;     // no line shared by rows
}
static int norm_entry(const char* who, NormRowArgs& a, int type, int sum_type, bool e4m3, void* stream) {
    VC_CHECK(check_norm(who, a.rows, a.cols, type, sum_type));
    if (a.rows == 0) return 0;
    VC_ARG(a.x && a.gamma && a.y && (!a.res || a.sum), "%s: null pointer", who);
    VC_ARG(a.eps > 0.f, "%s: eps must be positive", who);
    VC_CHECK(check_ld(who, a, {a.x_ld, a.res ? a.res_ld : 0}, {a.y_ld, a.res ? a.sum_ld : a.cols}));
    VC_ARG(a.rows <= 1 || ((a.y != a.x || a.y_ld == a.x_ld) && (!a.res || a.sum != a.res || a.sum_ld == a.res_ld)), "%s: in place, but with another row stride", who);
    VC_ARG(!e4m3 || a.y != a.x, "%s: q may not be x", who);
    if (!a.res) sum_type = type;
    const bool wide = sum_type == VC_F32 && type != VC_F32;
    set_past(a, type, wide);
    return SEQ_TYPES(type, norm_fwd, a, wide, e4m3, (hipStream_t)stream);
}
extern "C" int vc_rms_norm_fwd(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, const float* gamma,
                               void* y, int64_t y_ld, void* sum, int64_t sum_ld, float* rstd, float eps,
                               int64_t rows, int cols, int type, int sum_type, void* stream) {
    NormRowArgs a{};
    a.x = x; a.x_ld = x_ld; a.res = residual; a.res_ld = res_ld; a.gamma = gamma; a.y = y; a.y_ld = y_ld; a.sum = sum; a.sum_ld = sum_ld;
    a.rstd = rstd; a.eps = eps; a.rows = rows; a.cols = cols;
    return norm_entry("vc_rms_norm_fwd", a, type, sum_type, false, stream);
}
extern "C" int vc_rms_norm_e4m3(const void* x, int64_t x_ld, const void* residual, int64_t res_ld, const float* gamma,
                                void* q, int64_t q_ld, float* scale, void* sum, int64_t sum_ld, float eps,
                                int64_t rows, int cols, int group, int type, int sum_type, void* stream) {
    VC_ARG(group == 0 || ((group == 32 || group == 64 || group == 128) && cols % group == 0), "vc_rms_norm_e4m3: group must be 0, 32, 64 or 128 and divide cols");
    VC_ARG(scale || rows == 0, "vc_rms_norm_e4m3: null pointer");
    NormRowArgs a{};
    a.x = x; a.x_ld = x_ld; a.res = residual; a.res_ld = res_ld; a.gamma = gamma; a.y = q; a.y_ld = q_ld; a.scale = scale; a.sum = sum; a.sum_ld = sum_ld;
    a.eps = eps; a.rows = rows; a.cols = cols; a.group = group;
    return norm_entry("vc_rms_norm_e4m3", a, type, sum_type, true, stream);
}
extern "C" int64_t vc_rms_norm_bwd_work(int64_t rows, int cols) {
    VC_CHECK(check_norm("vc_rms_norm_bwd_work", rows, cols, VC_F32, VC_F32));
    return (int64_t)std::max(norm_bwd_blocks(rows, cols, VC_F32), norm_bwd_blocks(rows, cols, VC_BF16)) * cols;
}
extern "C" int vc_rms_norm_bwd(const void* dy, int64_t dy_ld, const void* dsum, int64_t dsum_ld, const void* sum, int64_t sum_ld,
                               const float* rstd, const float* gamma, void* dx, int64_t dx_ld, void* dres, int64_t dres_ld, float* dgamma,
                               float* work, int64_t work_floats, int64_t rows, int cols, int type, int sum_type, void* stream) {
    VC_CHECK(check_norm("vc_rms_norm_bwd", rows, cols, type, sum_type));
    if (rows == 0) {
        VC_ARG(!dgamma, "vc_rms_norm_bwd: no rows to take dgamma from");
        return 0;
    }
    VC_ARG(dy && sum && rstd && gamma && (dx || dres || dgamma), "vc_rms_norm_bwd: null pointer");
    if (dgamma && (!work || work_floats < vc_rms_norm_bwd_work(rows, cols))) { vc_set_error("vc_rms_norm_bwd: work is too small"); return VC_E_NOMEM; }
    NormRowArgs a{};
    a.dy = dy; a.dy_ld = dy_ld; a.dsum = dsum; a.dsum_ld = dsum_ld; a.sum = (void*)sum; a.sum_ld = sum_ld; a.rstd = (float*)rstd; a.gamma = gamma;
    a.dx = dx; a.dx_ld = dx_ld; a.dres = dres; a.dres_ld = dres_ld; a.rows = rows; a.cols = cols; a.part = dgamma ? work : nullptr;
    VC_CHECK(check_ld("vc_rms_norm_bwd", a, {dy_ld, dsum ? dsum_ld : 0, sum_ld}, {dx ? dx_ld : cols, dres ? dres_ld : cols}));
    const bool wide = sum_type == VC_F32 && type != VC_F32;
    set_past(a, type, wide);
    return SEQ_TYPES(type, norm_bwd, a, wide, type, dgamma, (hipStream_t)stream);
}

extern "C" int vc_seq_version(void) { return 1; }
