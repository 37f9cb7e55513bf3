// vc_seq_scan.hip -- selective state space scan: prompts and single frames (vc_seq_scan.h says how the work is laid out).
#include "vc_seq_scan.h"

constexpr int FWD_WAVES = 4;

// First pass of a split axis: what each run hands on.  Only rows from the last utterance's beginning on matter.  Bound by vector issue: a product, an
// exponential and two multiply-adds a state; 1 x 8192 x 1024 bf16, 16 states: 39 us, the main pass 54.
template <class T, int L, int NS> __global__ __launch_bounds__(256) void scan_edge_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L;
    __shared__ float lds[FWD_WAVES][TILE * NP];
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, item = blockIdx.x / nblk, blk = blockIdx.x - item * nblk;
    const Lane<L, NS> w(k, k.waves, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    const Rows<T, L> X(a.x, a.x_ld, a.cols, c, j), DT(a.dt, a.dt_ld, a.cols, c, j);
    const States<T, NP> B(a.B, a.b_ld, w.g, a.states, w.lane);
    float A2[NS], h[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn, w.full);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; h[i] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    int q0, q1;
    item_slots(k, item, q0, q1);
    Cursor cur(k.m);
    cur.find(q1 - 1);
    const bool cut = cur.base >= q0;                             // an utterance begins in this run
    if (cut && a.initial) load_state<NS>(a.initial + ((int64_t)cur.s * a.cols + c) * a.states + n0, h, nn, w.full);
    float* Bs = lds[w.wave];
    float sd = 0.f;
    const int k0 = max(q0 - cur.base, 0), k1 = min(cur.tiles, q1 - cur.base);
    T xr[NB], tr[NB], br[NP / 4];
    auto fetch = [&](int kt) {
        const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
        X.load(row0, nr, xr); DT.load(row0, nr, tr); B.load(row0, nr, br);
    };
    if (k0 < k1) fetch(k0);
    for (int kt = k0; kt < k1; ++kt) {
        const int nr = min(TILE, cur.end - cur.begin - kt * TILE);
        B.stage(br, nr, Bs);
        float delta[NB], dtx[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float slope;
            const float v = (float)tr[b] + bias, d = a.softplus ? softplus(v, slope) : v;
            delta[b] = b * L + j < nr ? d : 0.f;
            dtx[b] = b * L + j < nr ? d * (float)xr[b] : 0.f;
            sd += delta[b];
        }
        if (kt + 1 < k1) fetch(kt + 1);
        wave_lds_fence();
        static_for<0, NB>([&](auto b) {
            static_for<0, L>([&](auto i) {
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtx[b]);
                const float* Br = Bs + (b * L + i) * NP + n0;
#pragma unroll
                for (int e = 0; e < NS; ++e) h[e] = fmaf(exp2_fast(dl * A2[e]), h[e], dx * Br[e]);
            });
        });
        wave_lds_fence();
    }
    sd = channel_sum<L>(sd);
    if (w.ok) {
        store_state<NS>(k.edge + ((int64_t)item * a.cols + c) * a.states + n0, h, nn, w.full);
        if (j == 0) k.sum_delta[(int64_t)item * a.cols + c] = sd;
    }
    if (blk == 0 && threadIdx.x == 0) k.cut[item] = cut;
}

// Second pass of a split axis: from what every run hands on to what enters it, for 16 states a block.  SEGS threads share a state's runs: each goes through
// its own as if nothing entered them, what they do together -- h -> exp2(p) h + e, or e behind a cut -- is combined over the threads before, and each
// goes through its own once more from there.  A launch and a few trips to memory: 4 to 8 us, where one thread a state took 15 for 109 runs.  Up to 128 runs
// 16 threads are enough (2208 x 1002 x 12: 4 us less than by 64), for 425 runs they cost 8 us more.
constexpr int CARRY_W = 16;
template <int SEGS> __global__ __launch_bounds__(CARRY_W * SEGS) void scan_carry_kernel(const ScanK k, bool forward) {
    constexpr int KEEP = 8;
    __shared__ float ps[SEGS][CARRY_W], es[SEGS][CARRY_W];
    __shared__ int cs[SEGS][CARRY_W];
    const vc_scan_args& a = k.a;
    const int x = threadIdx.x % CARRY_W, seg = threadIdx.x / CARRY_W;
    const int64_t n = (int64_t)a.cols * a.states, at = (int64_t)blockIdx.x * CARRY_W + x, i = min(at, n - 1);      // past the last state: the last one again, not stored
    const int c = (int)(i / a.states), each = (k.items + SEGS - 1) / SEGS, first = min(seg * each, k.items), last = min(first + each, k.items);
    const float A2 = a.A[i] * LOG2E;
    float e[KEEP], p[KEEP]; int cut[KEEP];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            const int q = min(r0 + u, k.items - 1), r = forward ? q : k.items - 1 - q;
            e[u] = k.edge[r * n + i]; p[u] = A2 * k.sum_delta[(int64_t)r * a.cols + c]; cut[u] = k.cut[r];
        }
    };
    float h = 0.f, sum = 0.f; int any = 0;
    for (int r0 = first; r0 < last; r0 += KEEP) {
        fetch(r0);
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            if (r0 + u >= last) break;
            h = carried(p[u], h, e[u], cut[u]); sum += p[u]; any |= cut[u];
        }
    }
    ps[seg][x] = sum; es[seg][x] = h; cs[seg][x] = any;
    __syncthreads();
    for (int d = 1; d < SEGS; d *= 2) {
        const int b = max(seg - d, 0);
        const float pb = ps[b][x], eb = es[b][x]; const int cb = cs[b][x];
        __syncthreads();
        if (seg >= d) {
            h = carried(sum, eb, h, any); sum += pb; any |= cb;
            ps[seg][x] = sum; es[seg][x] = h; cs[seg][x] = any;
        }
        __syncthreads();
    }
    h = seg ? es[seg - 1][x] : 0.f;
    for (int r0 = first; r0 < last; r0 += KEEP) {
        if (last - first > KEEP) fetch(r0);
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            if (r0 + u >= last) break;
            if (at < n) k.edge[(forward ? r0 + u : k.items - 1 - r0 - u) * n + i] = h;
            h = carried(p[u], h, e[u], cut[u]);
        }
    }
}
int scan_carry(const ScanK& k, bool forward, hipStream_t s) {
    if (!k.once) return 0;
    const dim3 grid((unsigned)(((int64_t)k.a.cols * k.a.states + CARRY_W - 1) / CARRY_W));
    if (k.items <= 128) hipLaunchKernelGGL(scan_carry_kernel<16>, grid, dim3(CARRY_W * 16), 0, s, k, forward);
    else hipLaunchKernelGGL(scan_carry_kernel<64>, grid, dim3(CARRY_W * 64), 0, s, k, forward);
    VC_HIP(hipGetLastError());
    return 0;
}

template <int NS> struct RowPair {                                // B and C of two rows, a lane's states
    float b[2][NS], c[2][NS];
    __device__ __forceinline__ void read(const float* pb, const float* pc, int stride) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < NS; ++e) { b[u][e] = pb[u * stride + e]; c[u][e] = pc[u * stride + e]; }
    }
};

// One block walks the slots of one item for its waves * 64 / L channels.  The next tile's rows are on their way while a tile is worked on.
// Bound by vector issue: a row and channel costs a lane a product, an exponential (two slots) and three multiply-adds for each of its states, and its share
// of softplus, gate and sums.  64 x 128 x 1024 bf16, 16 states: 52 us with the vector units busy 85 % of the time (the bytes alone would take 14).
template <class T, int L, int NS> __global__ __launch_bounds__(256) void scan_fwd_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L;
    __shared__ float lds[FWD_WAVES][2][TILE * NP];
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, item = blockIdx.x / nblk, blk = blockIdx.x - item * nblk;
    const Lane<L, NS> w(k, k.waves, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    const Rows<T, L> Y(a.y, a.y_ld, a.cols, c, j, w.ok);
    if (item == k.items) {                                       // rows ahead of the first utterance and behind the last one
        Y.clear(0, seq_head(k.m), c, j);
        Y.clear(seq_tail(k.m), k.m.rows, c, j);
        return;
    }
    const bool has_z = a.z != nullptr;
    const Rows<T, L> X(a.x, a.x_ld, a.cols, c, j), DT(a.dt, a.dt_ld, a.cols, c, j), Z(has_z ? a.z : a.x, has_z ? a.z_ld : a.x_ld, a.cols, c, j);
    const States<T, NP> B(a.B, a.b_ld, w.g, a.states, w.lane), C(a.C, a.c_ld, w.g, a.states, w.lane);
    float A2[NS], h[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn, w.full);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; h[i] = 0.f; }
    const float Dc = a.D ? a.D[c] : 0.f, bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    int q0, q1;
    item_slots(k, item, q0, q1);
    Cursor cur(k.m);
    if (k.chunk) cur.find(q0); else cur.load(item);
    if (k.chunk && q0 > cur.base) carry_in<NS, true>(k, item, c, n0, nn, w.full, A2, h);
    float *Bs = lds[w.wave][0], *Cs = lds[w.wave][1];
    for (int q = q0; q < q1;) {                                  // the utterances of the item
        const int64_t hs = ((int64_t)cur.s * a.cols + c) * a.states + n0;
        const int k0 = max(q - cur.base, 0), k1 = min(cur.tiles, q1 - cur.base);
        const bool begins = q <= cur.base && cur.base < q1;      // (ahead of the first utterance lie slots of none)
        if (begins) {
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = 0.f;
            if (a.initial) load_state<NS>(a.initial + hs, h, nn, w.full);
        }
        T xr[NB], tr[NB], zr[NB], br[NP / 4], cr[NP / 4];
        auto fetch = [&](int kt) {
            const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
            X.load(row0, nr, xr); DT.load(row0, nr, tr);
            if (has_z) Z.load(row0, nr, zr);
            B.load(row0, nr, br); C.load(row0, nr, cr);
        };
        if (k0 < k1) fetch(k0);
        for (int kt = k0; kt < k1; ++kt) {
            const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
            if (a.saved && w.ok) store_state<NS>(a.saved + ((int64_t)(cur.base + kt) * a.cols + c) * a.states + n0, h, nn, w.full);
            B.stage(br, nr, Bs); C.stage(cr, nr, Cs);
            float delta[NB], dtx[NB], gate[NB], skip[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float slope;
                const float v = (float)tr[b] + bias, d = a.softplus ? softplus(v, slope) : v, xv = (float)xr[b];
                delta[b] = b * L + j < nr ? d : 0.f;
                dtx[b] = b * L + j < nr ? d * xv : 0.f;
                gate[b] = has_z ? (float)zr[b] * sigmoid<T>((float)zr[b]) : 1.f;
                skip[b] = Dc * xv;
            }
            if (kt + 1 < k1) fetch(kt + 1);
            const auto yt = Y.tile(row0, nr);
            wave_lds_fence();
            RowPair<NS> bc[2];
            bc[0].read(Bs + n0, Cs + n0, NP);
            static_for<0, NB>([&](auto b) {
                float acc[L];
                static_for<0, L / 2>([&](auto ii) {
                    constexpr int i = 2 * ii, t = b * L + i;
                    // the next two rows' B and C are fetched before these two are worked on; left alone, the scheduler asks for them when they are needed
                    if constexpr (t + 2 < TILE) bc[(t / 2 + 1) & 1].read(Bs + (t + 2) * NP + n0, Cs + (t + 2) * NP + n0, NP);
                    __builtin_amdgcn_sched_barrier(0);
                    const RowPair<NS>& r = bc[(t / 2) & 1];
                    const float dl[2] = {from_lane<L, i>(delta[b]), from_lane<L, i + 1>(delta[b])}, dx[2] = {from_lane<L, i>(dtx[b]), from_lane<L, i + 1>(dtx[b])};
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < NS; ++e) {
                            h[e] = fmaf(exp2_fast(dl[u] * A2[e]), h[e], dx[u] * r.b[u][e]);
                            sum = fmaf(r.c[u][e], h[e], sum);
                        }
                        acc[i + u] = sum;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                const float out = (sums_by_row<L>(acc, j) + skip[b]) * gate[b];
                Y.store(yt, b, out);
            });
            wave_lds_fence();
        }
        if (a.final_state && w.ok && (cur.tiles ? k0 < cur.tiles && k1 == cur.tiles : begins)) store_state<NS>(a.final_state + hs, h, nn, w.full);
        if (cur.next >= q1) break;
        q = max(cur.next, q + 1);
        cur.load(cur.s + 1);
    }
}

struct ScanStepArgs {
    const void *x, *dt, *z, *B, *C; const float *A, *D, *dt_bias; float* state; const int* slots; void* y;
    int64_t x_ld, dt_ld, z_ld, b_ld, c_ld, y_ld; int rows, n_slots, cols, states, groups, softplus; bool past;
};
// Bound by the state's traffic: L lanes a channel as in the scan, STEP_U channels a lane group.  Everything is asked for before the earlier rows' slots are
// looked through; a slot outside the pool reads entry 0 and drops it.  256 streams x 2048 bf16, 16 states: 16.3 us, 4.4 TB/s; one of 1024: 3.8 us.
constexpr int STEP_U = 2;
template <class T, int L, int NS> __global__ __launch_bounds__(256) void scan_step_kernel(const ScanStepArgs a) {
    constexpr int G = 256 / L;                                   // lane groups of a block
    const int r = blockIdx.y, j = threadIdx.x % L, c0 = blockIdx.x * (G * STEP_U) + threadIdx.x / L;
    const int mine = a.slots ? a.slots[r] : r, at = mine >= 0 && mine < a.n_slots ? mine : 0;
    const int n0 = j * NS, nn = max(0, min(NS, a.states - n0)), wide = a.cols / a.groups;
    const bool full = a.states == L * NS;                        // no lane lacks states: whole vectors without a question
    float h[STEP_U][NS], A[STEP_U][NS], B[STEP_U][NS], C[STEP_U][NS], x[STEP_U], z[STEP_U], v[STEP_U], D[STEP_U];
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) {
        const int c = min(c0 + u * G, a.cols - 1), g = c / wide;
        const float *hp = a.state + ((int64_t)at * a.cols + c) * a.states + n0, *ap = a.A + (int64_t)c * a.states + n0;
        const T *bp = (const T*)a.B + r * a.b_ld + g * a.states + n0, *cp = (const T*)a.C + r * a.c_ld + g * a.states + n0;
        load_state<NS>(hp, h[u], nn, full); load_state<NS>(ap, A[u], nn, full);
        if (full) { load_vec<T, NS>(bp, B[u]); load_vec<T, NS>(cp, C[u]); }
        else { load_some<T, NS>(bp, B[u], nn); load_some<T, NS>(cp, C[u], nn); }
        x[u] = (float)((const T*)a.x)[r * a.x_ld + c];
        v[u] = (float)((const T*)a.dt)[r * a.dt_ld + c] + (a.dt_bias ? a.dt_bias[c] : 0.f);
        z[u] = a.z ? (float)((const T*)a.z)[r * a.z_ld + c] : 0.f;
        D[u] = a.D ? a.D[c] : 0.f;
    }
    const bool padding = slot_is_padding(a.slots, r, mine, a.n_slots);
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) {
        const int c = c0 + u * G;
        if (c >= a.cols) break;
        T* y = (T*)a.y + (int64_t)r * a.y_ld + c;
        if (padding) { if (j == 0) *y = (T)0.f; continue; }
        float slope;
        const float d = a.softplus ? softplus(v[u], slope) : v[u];
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < NS; ++e) {
            h[u][e] = fmaf(exp2_fast(d * (A[u][e] * LOG2E)), h[u][e], d * x[u] * B[u][e]);
            sum = fmaf(C[u][e], h[u][e], sum);
        }
        float* hp = a.state + ((int64_t)mine * a.cols + c) * a.states + n0;
        store_out<float, NS>(hp, h[u], nn, a.past);
        sum = channel_sum<L>(sum) + D[u] * x[u];
        if (j == 0) *y = (T)(a.z ? sum * (z[u] * sigmoid<T>(z[u])) : sum);
    }
}

// Whole utterances, each walked by its own waves, or runs of slots, as many as make run_waves waves.  With w waves a SIMD side by side a row of the longest
// utterance takes about max(0.18, 0.1 w) us walked; in runs all rows are shared out, at 0.16 us a row for w = 1, since the first pass costs 0.7 of the main
// one, and the passes before the main one cost a few us more, the more waves the more (`margin`).  So walk where longest * (0.18 - 0.16 w) < 6 + margin w.
// Measured, bf16, 16 states, 1024 channels, forward (walked and in runs): 1 x 8192 frames 2880 and 103, 1 x 128 20 and 10, 1 x 32 6.9 and 9.1, 8 x 128 21
// and 27, 8 x 256 47 and 38, 16 x 512 91 and 102, 16 x 1024 194 and 185, 16 x 2048 400 and 338, 24 x 100 27 and 47, 64 x 128 54 and 94; the gradient 8 x 128 55 and 46, 16 x 512
// 214 and 210, 24 x 100 66 and 78, 1 x 32 the same.  1 x 8192 in runs for 1024 / 2048 / 4096 / 8192 waves: 162 / 112 / 103 / 103.  Few channels, training:
// 1 x 16384 x 64 82 in runs of a slot, 99 in runs of six.
constexpr int64_t FWD_RUN_WAVES = 4096;
constexpr double FWD_MARGIN = 14;
int scan_setup(const char* who, const vc_scan_args* a, int waves, int64_t run_waves, double margin, ScanK* k) {
    VC_ARG(a, "%s: null pointer", who);
    VC_ARG(seq_type_ok(a->type), "%s: type must be VC_F32, VC_BF16 or VC_F16", who);
    VC_ARG(a->states >= 1 && a->states <= 64, "%s: 1 to 64 states, got %d", who, a->states);
    VC_ARG(a->cols > 0 && a->groups > 0 && a->cols % a->groups == 0, "%s: groups (%d) must divide cols (%d)", who, a->groups, a->cols);
    VC_ARG(a->rows >= 0 && a->n_seqs > 0 && a->rows + (int64_t)TILE * a->n_seqs < (1LL << 31), "%s: bad sizes (rows %lld, n_seqs %d)", who, (long long)a->rows, a->n_seqs);
    VC_ARG(a->offsets || a->rows % a->n_seqs == 0, "%s: without offsets the rows divide into n_seqs equal utterances", who);
    for (int64_t ld : {a->x_ld, a->dt_ld, a->z ? a->z_ld : 0, a->b_ld, a->c_ld, a->y && a->rows > 1 ? a->y_ld : 0, a->dy ? a->dy_ld : 0})
        VC_ARG(ld >= 0 && ld <= MAX_LD && a->cols <= SEQ_COLS, "%s: row strides lie between 0 and 2^24 elements", who);
    if (a->rows > 1) {
        VC_ARG(!a->y || a->y_ld >= a->cols, "%s: rows of y overlap", who);
        VC_ARG(!a->dx || (a->dx_ld >= a->cols && a->dx_ld <= MAX_LD && a->ddt_ld >= a->cols && a->ddt_ld <= MAX_LD), "%s: row strides of dx and ddt lie between cols and 2^24", who);
        VC_ARG(!a->dz || (a->dz_ld >= a->cols && a->dz_ld <= MAX_LD), "%s: row strides of dz lie between cols and 2^24", who);
        VC_ARG(!a->dB || std::min(a->db_ld, a->dc_ld) >= (int64_t)a->groups * a->states, "%s: rows of dB or dC overlap", who);
    }
    *k = ScanK{};
    k->a = *a;
    // one row has no stride: the rows that its tile lacks are to lie behind it all the same, so that what is stored to them is dropped
    if (a->rows == 1) k->a.y_ld = k->a.dx_ld = k->a.ddt_ld = k->a.dz_ld = a->cols;
    k->m = SeqMap{a->offsets, (int)a->rows, a->n_seqs, (int)(a->rows / a->n_seqs)};
    k->cg = a->cols / a->groups;
    k->slots = (int)(a->rows / TILE) + a->n_seqs;
    const int cw = 64 / scan_lanes(a->states), need = (k->cg + cw - 1) / cw;     // channels of a wave; waves that a group's channels fill
    k->nblk = (need + waves - 1) / waves;
    k->waves = (need + k->nblk - 1) / k->nblk;                   // no wave without a channel, but for the last block's
    const int64_t row_waves = (int64_t)a->groups * need;         // waves that a frame's channels fill
    const int64_t longest = !a->offsets ? k->m.len : a->max_len > 0 ? a->max_len : a->rows;
    // utterances that run side by side for as long as the longest lasts
    const int64_t side = longest > 0 ? std::max<int64_t>(1, a->rows / longest) : a->n_seqs;
    k->items = a->n_seqs; k->chunk = 0;
    const int64_t want = std::max<int64_t>(1, run_waves / row_waves);
    // ... and runs where utterances are many and short: their first pass then has little to do, and the sums over items stay few
    const double w = side * row_waves / 1024.0;                  // waves a SIMD, walked
    const bool walk = longest * (0.18 - 0.16 * w) < 6 + margin * w;
    if (!walk || a->n_seqs > 4 * want) {
        k->chunk = (int)((k->slots + want - 1) / want);
        k->items = (k->slots + k->chunk - 1) / k->chunk;
        if (k->items == 1) { k->items = a->n_seqs; k->chunk = 0; }
        k->once = k->items > CARRY_ITEMS;
    }
    return 0;
}
int64_t scan_edge_floats(const ScanK& k) { return k.chunk ? (int64_t)k.items * ((int64_t)k.a.cols * (k.a.states + 1) + 1) : 0; }
void scan_edge_place(ScanK* k, float* work) {
    k->edge = work;
    k->sum_delta = work + (int64_t)k->items * k->a.cols * k->a.states;
    k->cut = (int*)(k->sum_delta + (int64_t)k->items * k->a.cols);
}
extern "C" int64_t vc_selective_scan_saved(const vc_scan_args* a) {
    ScanK k; if (scan_setup("vc_selective_scan_saved", a, FWD_WAVES, FWD_RUN_WAVES, FWD_MARGIN, &k)) return VC_E_ARG;
    return (int64_t)k.slots * a->cols * a->states;
}
extern "C" int64_t vc_selective_scan_fwd_work(const vc_scan_args* a) {
    ScanK k; if (scan_setup("vc_selective_scan_fwd_work", a, FWD_WAVES, FWD_RUN_WAVES, FWD_MARGIN, &k)) return VC_E_ARG;
    return scan_edge_floats(k);
}

template <class T, int L, int NS> static int scan_fwd_l(const ScanK& k, hipStream_t s) {
    const int64_t per = (int64_t)k.a.groups * k.nblk, blocks = per * (k.items + (k.a.zero_tail && k.m.off ? 1 : 0));
    VC_ARG(blocks < (1LL << 31), "vc_selective_scan_fwd: too many utterances and channels for one launch");
    if (k.chunk) {
        hipLaunchKernelGGL((scan_edge_kernel<T, L, NS>), dim3((unsigned)(per * k.items)), dim3(64 * k.waves), 0, s, k);
        VC_CHECK(scan_carry(k, true, s));
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS>), dim3((unsigned)blocks), dim3(64 * k.waves), 0, s, k);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int scan_fwd_t(const ScanK& k, hipStream_t s) { return SCAN_LAYOUT(T, k.a.states, scan_fwd_l, k, s); }
extern "C" int vc_selective_scan_fwd(const vc_scan_args* a, void* stream) {
    ScanK k; VC_CHECK(scan_setup("vc_selective_scan_fwd", a, FWD_WAVES, FWD_RUN_WAVES, FWD_MARGIN, &k));
    VC_ARG(a->A && (a->rows == 0 || (a->x && a->dt && a->B && a->C && a->y)), "vc_selective_scan_fwd: null pointer");
    VC_ARG(!a->final_state || a->final_state != a->initial, "vc_selective_scan_fwd: final_state may not be initial");
    if (a->saved && a->saved_floats < (int64_t)k.slots * a->cols * a->states) { vc_set_error("vc_selective_scan_fwd: saved is too small"); return VC_E_NOMEM; }
    if (scan_edge_floats(k) > 0 && (!a->work || a->work_floats < scan_edge_floats(k))) {
        vc_set_error("vc_selective_scan_fwd: work is too small (%lld floats needed)", (long long)scan_edge_floats(k));
        return VC_E_NOMEM;
    }
    if (k.chunk) scan_edge_place(&k, a->work);
    if (a->rows == 0 && !a->final_state) return 0;
    return SEQ_TYPES(a->type, scan_fwd_t, k, (hipStream_t)stream);
}

template <class T, int L, int NS> static int scan_step_l(const ScanStepArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((scan_step_kernel<T, L, NS>), dim3((a.cols + STEP_U * 256 / L - 1) / (STEP_U * 256 / L), a.rows), dim3(256), 0, s, a);
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
    VC_ARG(rows >= 0 && rows <= 65535 && n_slots > 0 && cols > 0 && cols <= SEQ_COLS && groups > 0 && cols % groups == 0,
           "vc_selective_scan_step: bad sizes (rows %d, n_slots %d, cols %d, groups %d)", rows, n_slots, cols, groups);
    VC_ARG(slots || rows <= n_slots, "vc_selective_scan_step: %d rows without slots, and %d slots", rows, n_slots);
    VC_ARG(!slots || rows <= MAX_SLOT_ROWS, "vc_selective_scan_step: at most %d rows with slots, got %d", MAX_SLOT_ROWS, rows);
    if (rows == 0) return 0;
    VC_ARG(x && dt && B && C && A && state && y, "vc_selective_scan_step: null pointer");
    VC_ARG(rows == 1 || (x_ld >= 0 && dt_ld >= 0 && (!z || z_ld >= 0) && b_ld >= 0 && c_ld >= 0 && y_ld >= cols), "vc_selective_scan_step: a row stride is out of range, or rows of y overlap");
    const ScanStepArgs a{x, dt, z, B, C, A, D, dt_bias, state, slots, y, x_ld, dt_ld, z_ld, b_ld, c_ld, y_ld, rows, n_slots, cols, states, groups, softplus, (int64_t)rows * cols * states * 4 >= STREAM_BYTES};
    return SEQ_TYPES(type, scan_step_t, a, (hipStream_t)stream);
}
