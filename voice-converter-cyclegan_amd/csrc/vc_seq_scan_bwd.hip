// vc_seq_scan_bwd.hip -- gradient of the selective state space scan (vc_seq_scan.h says how the work is laid out).
//   dh_t = C_t dp_t + a_{t+1} dh_{t+1} (dp = dy * gate, a = exp(delta A));  with q_t = dh_t a_t h_{t-1}:
//   dA = sum_t q delta;  ddelta = sum_n q A + x sum_n dh B;  dx = D dp + delta sum_n dh B;  dB = sum_c dh delta x;  dC = sum_c dp h
// A tile's states are worked out again from the one the forward kept in front of it: a and h of its 16 rows stay in registers for the way back.
#include "vc_seq_scan.h"

template <int L> constexpr int BWD_WAVES = L == 4 ? 8 : 4;      // LDS: B and C of each wave, and its share of dB and dC

// sum over the channels of a wave of its 2 NS values: the first steps hand one half of the values to the other half of the lanes.
template <int N> __device__ __forceinline__ void across_32(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + N / 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}
template <int N> __device__ __forceinline__ void across_16(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + N / 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}
// dst[i][64]: 2 NS = 8 values and L = 4: one a lane, item = bit3 + 2 bit4 + 4 bit5; 4 values: one a lane (the last channel steps not taken for L = 4),
// item = bit4 + 2 bit5; 8 values and L = 16: two a lane, item = i + 2 bit4 + 4 bit5
template <int L, int NS> __device__ __forceinline__ void reduce_to_lds(float (&v)[2 * NS], float* dst, int lane) {
    if constexpr (NS == 4) {
        float w[4], u[2];
        across_32<8>(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v[i];
        across_16<4>(w);
        u[0] = w[0]; u[1] = w[1];
        if constexpr (L == 4) {
            halve<0x128, 2>(u, lane & 8);
            dst[lane] = u[0];
        } else {
            dst[lane] = u[0]; dst[64 + lane] = u[1];
        }
    } else {
        float u[2];
        across_32<4>(v);
        u[0] = v[0]; u[1] = v[1];
        across_16<2>(u);
        dst[lane] = u[0];
    }
}
template <int L, int NS> constexpr int RED = (L == 16 && NS == 4) ? 128 : 64;      // floats a wave leaves for one row
// sum of item `it` (0..NS-1 dB, NS.. dC) of lane j of the channels, from what one wave left
template <int L, int NS> __device__ __forceinline__ float gather_item(const float* src, int it, int j) {
    if constexpr (L == 4 && NS == 4) {
        const int l = ((it & 1) << 3) + ((it & 2) << 3) + ((it & 4) << 3) + j;
        return src[l] + src[l + 4];
    } else if constexpr (L == 4) {
        const int l = ((it & 1) << 4) + ((it & 2) << 4) + j;
        return (src[l] + src[l + 4]) + (src[l + 8] + src[l + 12]);
    } else if constexpr (NS == 4) {
        return src[(it & 1) * 64 + ((it & 2) << 3) + ((it & 4) << 3) + j];
    } else {
        return src[((it & 1) << 4) + ((it & 2) << 4) + j];
    }
}

template <class T, int L, int NS> __global__ __launch_bounds__(64 * BWD_WAVES<L>, 1) void scan_bwd_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L, WV = BWD_WAVES<L>, R = RED<L, NS>;
    __shared__ float lds[WV][2][TILE * NP];
    __shared__ float red[WV][TILE * R];
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, s = blockIdx.x / nblk, blk = blockIdx.x - s * nblk;
    const Lane<L, NS> w(k, WV, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    T *dxo = (T*)a.dx + c, *ddt = (T*)a.ddt + c, *dzo = a.dz ? (T*)a.dz + c : nullptr;
    if (s == k.m.n_seqs) {
        if (w.ok)
            for (int r = seq_tail(k.m) + j; r < k.m.rows; r += L) {
                dxo[(int64_t)r * a.dx_ld] = (T)0.f; ddt[(int64_t)r * a.ddt_ld] = (T)0.f;
                if (dzo) dzo[(int64_t)r * a.dz_ld] = (T)0.f;
            }
        return;
    }
    const T *x = (const T*)a.x + c, *dt = (const T*)a.dt + c, *z = a.z ? (const T*)a.z + c : nullptr, *dy = (const T*)a.dy + c;
    const T *B = (const T*)a.B + w.g * a.states, *C = (const T*)a.C + w.g * a.states;
    float A2[NS], dA[NS], dhc[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; dA[i] = 0.f; dhc[i] = 0.f; }
    const float Dc = a.D ? a.D[c] : 0.f, bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    const int begin = seq_begin(k.m, s), end = seq_end(k.m, s, begin), base = slot_base(k.m, s);
    const int64_t hs = ((int64_t)s * a.cols + c) * a.states + n0;
    if (a.dfinal && w.ok) load_state<NS>(a.dfinal + hs, dhc, nn);
    float dDacc = 0.f, dbacc = 0.f;
    float *Bs = lds[w.wave][0], *Cs = lds[w.wave][1], *mine = red[w.wave];
    for (int kt = (end - begin + TILE - 1) / TILE - 1; kt >= 0; --kt) {
        const int row0 = begin + kt * TILE, nr = min(TILE, end - row0);
        stage_states<T, NP>(B, a.b_ld, row0, nr, a.states, Bs, w.lane);
        stage_states<T, NP>(C, a.c_ld, row0, nr, a.states, Cs, w.lane);
        float h0[NS];
        load_state<NS>(a.saved + ((int64_t)(base + kt) * a.cols + c) * a.states + n0, h0, nn);
        float xv[NB], delta[NB], slope[NB], dtx[NB], dp[NB], dzf[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const bool ok = w.ok && b * L + j < nr;
            const int64_t r = row0 + b * L + j;
            xv[b] = ok ? (float)x[r * a.x_ld] : 0.f;
            const float g = ok ? (float)dy[r * a.dy_ld] : 0.f, v = (ok ? (float)dt[r * a.dt_ld] : 0.f) + bias;
            slope[b] = 1.f;
            const float d = a.softplus ? softplus(v, slope[b]) : v;
            delta[b] = ok ? d : 0.f;
            dtx[b] = delta[b] * xv[b];
            dp[b] = g; dzf[b] = 0.f;
            if (z) {
                const float zv = ok ? (float)z[r * a.z_ld] : 0.f, sg = sigmoid_acc(zv);
                dp[b] = g * (zv * sg);
                dzf[b] = g * (sg * (1.f + zv * (1.f - sg)));
            }
        }
        wave_lds_fence();
        float av[TILE][NS], h[TILE][NS];
        static_for<0, NB>([&](auto b) {
            float acc[L];
            static_for<0, L>([&](auto i) {
                constexpr int t = b * L + i;
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtx[b]);
                const float *Br = Bs + t * NP + n0, *Cr = Cs + t * NP + n0;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    const float hp = t ? h[t ? t - 1 : 0][e] : h0[e];
                    av[t][e] = exp2_fast(dl * A2[e]);
                    h[t][e] = fmaf(av[t][e], hp, dx * Br[e]);
                    sum = fmaf(Cr[e], h[t][e], sum);
                }
                acc[i] = sum;
                __builtin_amdgcn_sched_barrier(0);      // B and C of later rows wait in LDS, not in registers: 128 of them hold a and h
            });
            if (dzo) {
                const float yp = sums_by_row<L>(acc, j) + Dc * xv[b];
                if (w.ok && b * L + j < nr) dzo[(int64_t)(row0 + b * L + j) * a.dz_ld] = (T)(dzf[b] * yp);
            }
        });
        static_for<0, NB>([&](auto bb) {
            constexpr int b = NB - 1 - bb;
            float gacc[L], qacc[L];
            static_for<0, L>([&](auto ii) {
                constexpr int i = L - 1 - ii, t = b * L + i;
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtx[b]), dpl = from_lane<L, i>(dp[b]);
                const float *Br = Bs + t * NP + n0, *Cr = Cs + t * NP + n0;
                float v[2 * NS], g = 0.f, qs = 0.f;
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    const float hp = t ? h[t ? t - 1 : 0][e] : h0[e];
                    const float dh = fmaf(dpl, Cr[e], dhc[e]);
                    v[NS + e] = dpl * h[t][e];
                    v[e] = dh * dx;
                    g = fmaf(dh, Br[e], g);
                    dhc[e] = av[t][e] * dh;
                    const float q = dhc[e] * hp;
                    qs = fmaf(q, A2[e], qs);
                    dA[e] = fmaf(q, dl, dA[e]);
                }
                gacc[i] = g; qacc[i] = qs;
                reduce_to_lds<L, NS>(v, mine + t * R, w.lane);
                __builtin_amdgcn_sched_barrier(0);
            });
            const float g = sums_by_row<L>(gacc, j), q = sums_by_row<L>(qacc, j) * LN2;
            const float dv = (q + xv[b] * g) * slope[b];
            dDacc = fmaf(dp[b], xv[b], dDacc);
            if (w.ok && b * L + j < nr) {
                dbacc += dv;
                const int64_t r = row0 + b * L + j;
                dxo[r * a.dx_ld] = (T)fmaf(delta[b], g, dp[b] * Dc);
                ddt[r * a.ddt_ld] = (T)dv;
            }
        });
        __syncthreads();
        for (int o = threadIdx.x; o < nr * 2 * NP; o += 64 * WV) {
            const int t = o / (2 * NP), e = o % (2 * NP), n = e % NP, it = (e / NP) * NS + n % NS;
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < WV; ++v) sum += gather_item<L, NS>(red[v] + t * R, it, n / NS);
            k.part[((int64_t)blk * k.m.rows + row0 + t) * (2 * NP) + e] = sum;
        }
        __syncthreads();
    }
    if (w.ok) {
        if (a.dinitial) store_some<float, NS>(a.dinitial + hs, dhc, nn);
        store_some<float, NS>(k.dapart + hs, dA, nn);
    }
    const float d = channel_sum<L>(dDacc), b = channel_sum<L>(dbacc);
    if (w.ok && j == 0) {
        k.chpart[((int64_t)s * 2) * a.cols + c] = d;
        k.chpart[((int64_t)s * 2 + 1) * a.cols + c] = b;
    }
}

// dB, dC: sum over the blocks of a group, rounded once
template <class T> __global__ __launch_bounds__(256) void scan_dbc_kernel(const ScanK k, int np) {
    const vc_scan_args& a = k.a;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int w = 2 * np * a.groups, tail = seq_tail(k.m);
    if (i >= (int64_t)k.m.rows * w) return;
    const int64_t r = i / w;
    const int e = (int)(i - r * w), g = e / (2 * np), m = e % (2 * np), n = m % np;
    if (n >= a.states) return;
    T* dst = m < np ? (T*)a.dB + r * a.db_ld : (T*)a.dC + r * a.dc_ld;
    dst += g * a.states + n;
    if (r >= tail) { if (a.zero_tail) *dst = (T)0.f; return; }
    float s = 0.f;
    for (int b = 0; b < k.nblk; ++b) s += k.part[((int64_t)(g * k.nblk + b) * k.m.rows + r) * (2 * np) + m];
    *dst = (T)s;
}
// dA, dD, ddt_bias: sum over the utterances
__global__ __launch_bounds__(256) void scan_param_kernel(const ScanK k, int items) {
    const vc_scan_args& a = k.a;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, na = (int64_t)a.cols * a.states;
    if (i < na) {
        float s = 0.f;
        for (int q = 0; q < items; ++q) s += k.dapart[q * na + i];
        a.dA[i] = s;
    } else if (i < na + 2 * a.cols) {
        const int64_t e = i - na;
        float* dst = e < a.cols ? a.dD : a.ddt_bias;
        if (!dst) return;
        float s = 0.f;
        for (int q = 0; q < items; ++q) s += k.chpart[(int64_t)q * 2 * a.cols + e];
        dst[e % a.cols] = s;
    }
}

static int bwd_setup(const char* who, const vc_scan_args* a, ScanK* k, int64_t* floats) {
    VC_CHECK(scan_setup(who, a, true, k));
    const int per = (scan_lanes(a->states) == 4 ? BWD_WAVES<4> : BWD_WAVES<16>) * 64 / scan_lanes(a->states);
    k->nblk = (k->cg + per - 1) / per;
    const int64_t part = (int64_t)a->groups * k->nblk * a->rows * 2 * scan_padded(a->states);
    const int64_t da = (int64_t)a->n_seqs * a->cols * a->states, ch = (int64_t)a->n_seqs * 2 * a->cols;
    *floats = part + da + ch;
    k->part = a->work; k->dapart = a->work + part; k->chpart = a->work + part + da;
    return 0;
}
extern "C" int64_t vc_selective_scan_bwd_work(const vc_scan_args* a) {
    ScanK k{}; int64_t n;
    return bwd_setup("vc_selective_scan_bwd_work", a, &k, &n) ? VC_E_ARG : n;
}
template <class T, int L, int NS> static int scan_bwd_l(const ScanK& k, hipStream_t s) {
    const int64_t blocks = (int64_t)k.a.groups * k.nblk * (k.m.n_seqs + (k.a.zero_tail && k.m.off ? 1 : 0));
    const int64_t bc = ((int64_t)k.m.rows * 2 * L * NS * k.a.groups + 255) / 256, pr = ((int64_t)k.a.cols * (k.a.states + 2) + 255) / 256;
    VC_ARG(blocks < (1LL << 31) && bc < (1LL << 31), "vc_selective_scan_bwd: too many utterances and channels for one launch");
    hipLaunchKernelGGL((scan_bwd_kernel<T, L, NS>), dim3((unsigned)blocks), dim3(64 * BWD_WAVES<L>), 0, s, k);
    if (bc) hipLaunchKernelGGL((scan_dbc_kernel<T>), dim3((unsigned)bc), dim3(256), 0, s, k, L * NS);
    hipLaunchKernelGGL(scan_param_kernel, dim3((unsigned)pr), dim3(256), 0, s, k, k.m.n_seqs);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int scan_bwd_t(const ScanK& k, hipStream_t s) { return SCAN_LAYOUT(T, k.a.states, scan_bwd_l, k, s); }
extern "C" int vc_selective_scan_bwd(const vc_scan_args* a, void* stream) {
    ScanK k{}; int64_t need;
    VC_CHECK(bwd_setup("vc_selective_scan_bwd", a, &k, &need));
    VC_ARG(a->A && a->dA && (a->rows == 0 || (a->x && a->dt && a->B && a->C && a->dy && a->dx && a->ddt && a->dB && a->dC && a->saved)), "vc_selective_scan_bwd: null pointer");
    VC_ARG(!a->z || a->dz, "vc_selective_scan_bwd: z has a gradient, dz is null");
    if (!a->z) k.a.dz = nullptr;
    if (a->saved_floats < vc_selective_scan_saved(a) && a->rows) { vc_set_error("vc_selective_scan_bwd: saved is too small"); return VC_E_NOMEM; }
    if (a->work_floats < need || !a->work) { vc_set_error("vc_selective_scan_bwd: work is too small (%lld floats needed)", (long long)need); return VC_E_NOMEM; }
    return SEQ_TYPES(a->type, scan_bwd_t, k, (hipStream_t)stream);
}
