// vc_seq_norm.hip -- RMS norm of a frame's channels with the residual's addition, its 8-bit form, its gradient.
//   t = x + residual (as stored);  y = t * rstd * gamma,  rstd = 1 / sqrt(mean(t^2) + eps)
#include "vc_seq.h"

struct NormRowArgs {
    const void* x; const void* res; const float* gamma; void* y; void* sum; float* rstd; float* scale;
    const void* dy; const void* dsum; void* dx; void* dres;
    int64_t x_ld, res_ld, y_ld, sum_ld, dy_ld, dsum_ld, dx_ld, dres_ld;
    float eps; int64_t rows; int cols, group;
};

template <class T, class S> __global__ __launch_bounds__(256) void rms_fwd_kernel(const NormRowArgs a) {
    __shared__ float red[4];
    const int64_t r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.x_ld;
    const S* res = a.res ? (const S*)a.res + r * a.res_ld : nullptr;
    S* sum = a.sum ? (S*)a.sum + r * a.sum_ld : nullptr;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float t = res ? (float)(S)((float)x[c] + (float)res[c]) : (float)x[c];
        ss += t * t;
    }
    ss = block_sum_256(ss, red);
    const float rstd = 1.f / sqrtf(ss / (float)a.cols + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float t = res ? (float)(S)((float)x[c] + (float)res[c]) : (float)x[c];
        if (sum && res) sum[c] = (S)t;
        ((T*)a.y)[r * a.y_ld + c] = (T)(t * rstd * a.gamma[c]);
    }
}
template <class T, class S> __global__ __launch_bounds__(256) void rms_e4m3_kernel(const NormRowArgs a) {
    __shared__ float red[4];
    __shared__ unsigned top;
    const int64_t r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.x_ld;
    const S* res = a.res ? (const S*)a.res + r * a.res_ld : nullptr;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float t = res ? (float)(S)((float)x[c] + (float)res[c]) : (float)x[c];
        ss += t * t;
    }
    ss = block_sum_256(ss, red);
    const float rstd = 1.f / sqrtf(ss / (float)a.cols + a.eps);
    const int w = a.group ? a.group : a.cols, ng = a.cols / w;
    for (int g = 0; g < ng; ++g) {
        __syncthreads();
        if (threadIdx.x == 0) top = __float_as_uint(0x1p-100f);
        __syncthreads();
        for (int c = g * w + threadIdx.x; c < (g + 1) * w; c += 256) {
            const float t = res ? (float)(S)((float)x[c] + (float)res[c]) : (float)x[c];
            atomicMax(&top, __float_as_uint(fabsf(t * rstd * a.gamma[c])));      // as integers: NaN is above infinity, and stays
        }
        __syncthreads();
        const float m = __uint_as_float(top);
        const float inv = 448.f / m;
        if (threadIdx.x == 0) a.scale[r * ng + g] = m / 448.f;
        for (int c = g * w + threadIdx.x; c < (g + 1) * w; c += 256) {
            const float t = res ? (float)(S)((float)x[c] + (float)res[c]) : (float)x[c];
            if (a.sum && res) ((S*)a.sum)[r * a.sum_ld + c] = (S)t;
            const float v = t * rstd * a.gamma[c] * inv;
            ((unsigned char*)a.y)[r * a.y_ld + c] = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false);
        }
    }
}
template <class T, class S> __global__ __launch_bounds__(256) void rms_bwd_kernel(const NormRowArgs a) {
    __shared__ float red[4];
    const int64_t r = blockIdx.x;
    const S* t = (const S*)a.sum + r * a.sum_ld;
    const T* dy = (const T*)a.dy + r * a.dy_ld;
    const S* ds = a.dsum ? (const S*)a.dsum + r * a.dsum_ld : nullptr;
    const float rstd = a.rstd[r];
    float m = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 256) m += (float)dy[c] * a.gamma[c] * ((float)t[c] * rstd);
    m = block_sum_256(m, red) / (float)a.cols;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        const float g = (float)dy[c] * a.gamma[c];
        const float d = (ds ? (float)ds[c] : 0.f) + rstd * (g - (float)t[c] * rstd * m);
        if (a.dx) ((T*)a.dx)[r * a.dx_ld + c] = (T)d;
        if (a.dres) ((S*)a.dres)[r * a.dres_ld + c] = (S)d;
    }
}
template <class T, class S> __global__ __launch_bounds__(64) void rms_dgamma_kernel(const NormRowArgs a, float* dgamma) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= a.cols) return;
    float s = 0.f;
    for (int64_t r = 0; r < a.rows; ++r) s += (float)((const T*)a.dy)[r * a.dy_ld + c] * ((float)((const S*)a.sum)[r * a.sum_ld + c] * a.rstd[r]);
    dgamma[c] = s;
}

template <class T, class S> static int norm_fwd_t(const NormRowArgs& a, bool e4m3, hipStream_t s) {
    if (e4m3) hipLaunchKernelGGL((rms_e4m3_kernel<T, S>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rms_fwd_kernel<T, S>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int norm_fwd(const NormRowArgs& a, bool wide, bool e4m3, hipStream_t s) {
    return wide ? norm_fwd_t<T, float>(a, e4m3, s) : norm_fwd_t<T, T>(a, e4m3, s);
}
template <class T, class S> static int norm_bwd_t(const NormRowArgs& a, float* dgamma, hipStream_t s) {
    if (a.dx || a.dres) hipLaunchKernelGGL((rms_bwd_kernel<T, S>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    if (dgamma) hipLaunchKernelGGL((rms_dgamma_kernel<T, S>), dim3((a.cols + 63) / 64), dim3(64), 0, s, a, dgamma);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int norm_bwd(const NormRowArgs& a, bool wide, float* dgamma, hipStream_t s) {
    return wide ? norm_bwd_t<T, float>(a, dgamma, s) : norm_bwd_t<T, T>(a, dgamma, s);
}

static int check_norm(const char* who, int64_t rows, int cols, int type, int sum_type) {
    VC_ARG(rows >= 0 && rows < (1LL << 31) && cols > 0, "%s: bad sizes (rows %lld, cols %d)", who, (long long)rows, cols);
    VC_ARG(seq_type_ok(type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(sum_type == type || sum_type == VC_F32, "%s: the residual stream has the activations' type or fp32", who);
    return 0;
}
static int norm_entry(const char* who, NormRowArgs& a, int type, int sum_type, bool e4m3, void* stream) {
    VC_CHECK(check_norm(who, a.rows, a.cols, type, sum_type));
    if (a.rows == 0) return 0;
    VC_ARG(a.x && a.gamma && a.y && (!a.res || a.sum), "%s: null pointer", who);
    VC_ARG(a.eps > 0.f, "%s: eps must be positive", who);
    if (!a.res) sum_type = type;
    const bool wide = sum_type == VC_F32 && type != VC_F32;
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
extern "C" int64_t vc_rms_norm_bwd_work(int64_t rows, int cols) { return 0; }
extern "C" int vc_rms_norm_bwd(const void* dy, int64_t dy_ld, const void* dsum, int64_t dsum_ld, const void* sum, int64_t sum_ld,
                               const float* rstd, const float* gamma, void* dx, int64_t dx_ld, void* dres, int64_t dres_ld, float* dgamma,
                               float* work, int64_t work_floats, int64_t rows, int cols, int type, int sum_type, void* stream) {
    VC_CHECK(check_norm("vc_rms_norm_bwd", rows, cols, type, sum_type));
    if (rows == 0) {
        VC_ARG(!dgamma, "vc_rms_norm_bwd: no rows to take dgamma from");
        return 0;
    }
    VC_ARG(dy && sum && rstd && gamma && (dx || dres || dgamma), "vc_rms_norm_bwd: null pointer");
    NormRowArgs a{};
    a.dy = dy; a.dy_ld = dy_ld; a.dsum = dsum; a.dsum_ld = dsum_ld; a.sum = (void*)sum; a.sum_ld = sum_ld; a.rstd = (float*)rstd; a.gamma = gamma;
    a.dx = dx; a.dx_ld = dx_ld; a.dres = dres; a.dres_ld = dres_ld; a.rows = rows; a.cols = cols;
    return SEQ_TYPES(type, norm_bwd, a, sum_type == VC_F32 && type != VC_F32, dgamma, (hipStream_t)stream);
}

extern "C" int vc_seq_version(void) { return 1; }
