// vc_seq_scan.hip -- selective state space scan: prompts and single frames (vc_seq_scan.h says how the work is laid out).
#include "vc_seq_scan.h"

constexpr int FWD_WAVES = 4;

// One block walks one utterance for FWD_WAVES * 64 / L channels, tile by tile.
template <class T, int L, int NS> __global__ __launch_bounds__(256) void scan_fwd_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L;
    __shared__ float lds[FWD_WAVES][2][TILE * NP];
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, s = blockIdx.x / nblk, blk = blockIdx.x - s * nblk;
    const Lane<L, NS> w(k, FWD_WAVES, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    const T *x = (const T*)a.x + c, *dt = (const T*)a.dt + c, *z = a.z ? (const T*)a.z + c : nullptr;
    const T *B = (const T*)a.B + w.g * a.states, *C = (const T*)a.C + w.g * a.states;
    T* y = (T*)a.y + c;
    if (s == k.m.n_seqs) {                                       // rows behind the last utterance
        if (w.ok) for (int r = seq_tail(k.m) + j; r < k.m.rows; r += L) y[(int64_t)r * a.y_ld] = (T)0.f;
        return;
    }
    float A2[NS], h[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; h[i] = 0.f; }
    const float Dc = a.D ? a.D[c] : 0.f, bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    const int begin = seq_begin(k.m, s), end = seq_end(k.m, s, begin), base = slot_base(k.m, s);
    const int64_t hs = ((int64_t)s * a.cols + c) * a.states + n0;
    if (a.initial) load_state<NS>(a.initial + hs, h, nn);
    float *Bs = lds[w.wave][0], *Cs = lds[w.wave][1];
    for (int row0 = begin, q = base; row0 < end; row0 += TILE, ++q) {
        const int nr = min(TILE, end - row0);
        if (a.saved && w.ok) store_some<float, NS>(a.saved + ((int64_t)q * a.cols + c) * a.states + n0, h, nn);
        stage_states<T, NP>(B, a.b_ld, row0, nr, a.states, Bs, w.lane);
        stage_states<T, NP>(C, a.c_ld, row0, nr, a.states, Cs, w.lane);
        float delta[NB], dtx[NB], gate[NB], skip[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const bool ok = b * L + j < nr;
            const int64_t r = row0 + b * L + j;
            const float xv = ok ? (float)x[r * a.x_ld] : 0.f, zv = ok && z ? (float)z[r * a.z_ld] : 0.f;
            const float v = (ok ? (float)dt[r * a.dt_ld] : 0.f) + bias;
            float slope;
            const float d = a.softplus ? softplus(v, slope) : v;
            delta[b] = ok ? d : 0.f;
            dtx[b] = delta[b] * xv;
            gate[b] = z ? zv * sigmoid_acc(zv) : 1.f;
            skip[b] = Dc * xv;
        }
        wave_lds_fence();
        static_for<0, NB>([&](auto b) {
            float acc[L];
            static_for<0, L>([&](auto i) {
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtx[b]);
                const float *Br = Bs + (b * L + i) * NP + n0, *Cr = Cs + (b * L + i) * NP + n0;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    h[e] = fmaf(exp2_fast(dl * A2[e]), h[e], dx * Br[e]);
                    sum = fmaf(Cr[e], h[e], sum);
                }
                acc[i] = sum;
            });
            const float out = (sums_by_row<L>(acc, j) + skip[b]) * gate[b];
            if (w.ok && b * L + j < nr) y[(int64_t)(row0 + b * L + j) * a.y_ld] = (T)out;
        });
        wave_lds_fence();
    }
    if (a.final_state && w.ok) store_some<float, NS>(a.final_state + hs, h, nn);
}

struct ScanStepArgs {
    const void *x, *dt, *z, *B, *C; const float *A, *D, *dt_bias; float* state; const int* slots; void* y;
    int64_t x_ld, dt_ld, z_ld, b_ld, c_ld, y_ld; int rows, n_slots, cols, states, groups, softplus;
};
template <class T, int L, int NS> __global__ __launch_bounds__(256) void scan_step_kernel(const ScanStepArgs a) {
    const int r = blockIdx.y, j = threadIdx.x % L, c = blockIdx.x * (256 / L) + threadIdx.x / L;
    const int slot = claim_slot(a.slots, r, a.n_slots);
    if (c >= a.cols) return;
    T* y = (T*)a.y + (int64_t)r * a.y_ld + c;
    if (slot < 0) { if (j == 0) *y = (T)0.f; return; }
    const int n0 = j * NS, nn = max(0, min(NS, a.states - n0)), g = c / (a.cols / a.groups);
    float* st = a.state + ((int64_t)slot * a.cols + c) * a.states + n0;
    float h[NS], A[NS], B[NS], C[NS];
    load_state<NS>(st, h, nn);
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A, nn);
    load_some<T, NS>((const T*)a.B + r * a.b_ld + g * a.states + n0, B, nn);
    load_some<T, NS>((const T*)a.C + r * a.c_ld + g * a.states + n0, C, nn);
    const float x = (float)((const T*)a.x)[r * a.x_ld + c], z = a.z ? (float)((const T*)a.z)[r * a.z_ld + c] : 0.f;
    const float v = (float)((const T*)a.dt)[r * a.dt_ld + c] + (a.dt_bias ? a.dt_bias[c] : 0.f);
    float slope;
    const float d = a.softplus ? softplus(v, slope) : v;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < NS; ++e) {
        h[e] = fmaf(exp2_fast(d * (A[e] * LOG2E)), h[e], d * x * B[e]);
        sum = fmaf(C[e], h[e], sum);
    }
    store_some<float, NS>(st, h, nn);
    sum = channel_sum<L>(sum) + (a.D ? a.D[c] * x : 0.f);
    if (j == 0) *y = (T)(a.z ? sum * (z * sigmoid_acc(z)) : sum);
}

int scan_setup(const char* who, const vc_scan_args* a, bool bwd, ScanK* k) {
    VC_ARG(a, "%s: null pointer", who);
    VC_ARG(seq_type_ok(a->type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(a->states >= 1 && a->states <= 64, "%s: 1 to 64 states, got %d", who, a->states);
    VC_ARG(a->cols > 0 && a->groups > 0 && a->cols % a->groups == 0, "%s: groups (%d) must divide cols (%d)", who, a->groups, a->cols);
    VC_ARG(a->rows >= 0 && a->n_seqs > 0 && a->rows + (int64_t)TILE * a->n_seqs < (1LL << 31), "%s: bad sizes (rows %lld, n_seqs %d)", who, (long long)a->rows, a->n_seqs);
    VC_ARG(a->offsets || a->rows % a->n_seqs == 0, "%s: without offsets the rows divide into n_seqs equal utterances", who);
    k->a = *a;
    k->m = SeqMap{a->offsets, (int)a->rows, a->n_seqs, (int)(a->rows / a->n_seqs)};
    k->cg = a->cols / a->groups;
    k->slots = (int)(a->rows / TILE) + a->n_seqs;
    return 0;
}
extern "C" int64_t vc_selective_scan_saved(const vc_scan_args* a) {
    ScanK k; if (scan_setup("vc_selective_scan_saved", a, false, &k)) return VC_E_ARG;
    return (int64_t)k.slots * a->cols * a->states;
}
extern "C" int64_t vc_selective_scan_fwd_work(const vc_scan_args* a) { ScanK k; return scan_setup("vc_selective_scan_fwd_work", a, false, &k) ? VC_E_ARG : 0; }

template <class T, int L, int NS> static int scan_fwd_l(const ScanK& k, hipStream_t s) {
    const int64_t blocks = (int64_t)k.a.groups * k.nblk * (k.m.n_seqs + (k.a.zero_tail && k.m.off ? 1 : 0));
    VC_ARG(blocks < (1LL << 31), "vc_selective_scan_fwd: too many utterances and channels for one launch");
    hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS>), dim3((unsigned)blocks), dim3(64 * FWD_WAVES), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int scan_fwd_t(const ScanK& k, hipStream_t s) { return SCAN_LAYOUT(T, k.a.states, scan_fwd_l, k, s); }
extern "C" int vc_selective_scan_fwd(const vc_scan_args* a, void* stream) {
    ScanK k{}; VC_CHECK(scan_setup("vc_selective_scan_fwd", a, false, &k));
    VC_ARG(a->A && (a->rows == 0 || (a->x && a->dt && a->B && a->C && a->y)), "vc_selective_scan_fwd: null pointer");
    VC_ARG(!a->final_state || a->final_state != a->initial, "vc_selective_scan_fwd: final_state may not be initial");
    if (a->saved && a->saved_floats < vc_selective_scan_saved(a)) { vc_set_error("vc_selective_scan_fwd: saved is too small"); return VC_E_NOMEM; }
    if (a->rows == 0 && !a->final_state) return 0;
    const int per = FWD_WAVES * 64 / scan_lanes(a->states);
    k.nblk = (k.cg + per - 1) / per;
    return SEQ_TYPES(a->type, scan_fwd_t, k, (hipStream_t)stream);
}

template <class T, int L, int NS> static int scan_step_l(const ScanStepArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((scan_step_kernel<T, L, NS>), dim3((a.cols + 256 / L - 1) / (256 / L), a.rows), dim3(256), 0, s, a);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int scan_step_t(const ScanStepArgs& a, hipStream_t s) { return SCAN_LAYOUT(T, a.states, scan_step_l, a, s); }
extern "C" int vc_selective_scan_step(const void* x, int64_t x_ld, const void* dt, int64_t dt_ld, const void* z, int64_t z_ld,
                                      const void* B, int64_t b_ld, const void* C, int64_t c_ld, const float* A, const float* D, const float* dt_bias,
                                      float* state, const int32_t* slots, void* y, int64_t y_ld,
                                      int rows, int n_slots, int cols, int states, int groups, int type, int softplus, void* stream) {
    VC_ARG(seq_type_ok(type), "vc_selective_scan_step: type must be VC_F32, VC_BF16 or VC_F16");
    VC_ARG(states >= 1 && states <= 64, "vc_selective_scan_step: 1 to 64 states, got %d", states);
    VC_ARG(rows >= 0 && rows <= 65535 && n_slots > 0 && cols > 0 && groups > 0 && cols % groups == 0,
           "vc_selective_scan_step: bad sizes (rows %d, n_slots %d, cols %d, groups %d)", rows, n_slots, cols, groups);
    VC_ARG(slots || rows <= n_slots, "vc_selective_scan_step: %d rows without slots, and %d slots", rows, n_slots);
    if (rows == 0) return 0;
    VC_ARG(x && dt && B && C && A && state && y, "vc_selective_scan_step: null pointer");
    const ScanStepArgs a{x, dt, z, B, C, A, D, dt_bias, state, slots, y, x_ld, dt_ld, z_ld, b_ld, c_ld, y_ld, rows, n_slots, cols, states, groups, softplus};
    return SEQ_TYPES(type, scan_step_t, a, (hipStream_t)stream);
}
