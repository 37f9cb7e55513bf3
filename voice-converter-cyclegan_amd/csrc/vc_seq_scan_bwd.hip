// vc_seq_scan_bwd.hip -- gradient of the selective state space scan (vc_seq_scan.h says how the work is laid out).
//   dh_t = C_t dp_t + a_{t+1} dh_{t+1} (dp = dy * gate, a = exp(delta A));  with q_t = dh_t a_t h_{t-1}:
//   dA = sum_t q delta;  ddelta = sum_n q A + x sum_n dh B;  dx = D dp + delta sum_n dh B;  dB = sum_c dh delta x;  dC = sum_c dp h
// A tile's states are worked out again from the one the forward kept in front of it: a and h of its 16 rows stay in registers for the way back.
// Bound by vector issue: six slots a state on the way there, eight and five for the sums over channels on the way back, two waves a SIMD (the registers).
// 64 x 128 x 1024 bf16, 16 states: 136 us, the vector units busy 83 % of the time.
#include "vc_seq_scan.h"

constexpr int BWD_WAVES = 4;                                     // of a block.  8 leave half as many partial sums of dB and dC and cost 2 %: more waves stand at a barrier together

template <int NS> struct Row {                                    // B and C of a row, a lane's states
    float b[NS], c[NS];
    __device__ __forceinline__ void read(const float* pb, const float* pc) {
#pragma unroll
        for (int e = 0; e < NS; ++e) { b[e] = pb[e]; c[e] = pc[e]; }
    }
};
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
// dst[i][64]: 2 NS = 8 values and L = 4 or 8: one a lane, item = bit3 + 2 bit4 + 4 bit5; 4 values: one a lane (the last channel steps not taken for L = 4),
// item = bit4 + 2 bit5; 8 values and L = 16: two a lane, item = i + 2 bit4 + 4 bit5
template <int L, int NS> __device__ __forceinline__ void reduce_to_lds(float (&v)[2 * NS], float* dst, int lane) {
    if constexpr (NS == 4) {
        float w[4], u[2];
        across_32<8>(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v[i];
        across_16<4>(w);
        u[0] = w[0]; u[1] = w[1];
        if constexpr (L <= 8) {
            halve<0x128, 2>(u, lane & 8);                        // row_ror:8
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
// what one wave left of item `it` (0..NS-1 dB, NS.. dC) of lane j of the channels: SPLIT numbers to be added
template <int L, int NS> constexpr int SPLIT = L >= 8 ? 1 : NS == 4 ? 2 : 4;
template <int L, int NS> __device__ __forceinline__ int item_at(int it, int j) {
    if constexpr (L <= 8 && NS == 4) return ((it & 1) << 3) + ((it & 2) << 3) + ((it & 4) << 3) + j;
    else if constexpr (NS == 4) return (it & 1) * 64 + ((it & 2) << 3) + ((it & 4) << 3) + j;
    else return ((it & 1) << 4) + ((it & 2) << 4) + j;
}

// First pass of a split axis: what each run hands on to the one before it.  Only rows up to the end of the run's first utterance matter.  Bound by vector
// issue, like the forward's; 2208 x 1002 fp32, 12 states: 16 us.
template <class T, int L, int NS> __global__ __launch_bounds__(64 * BWD_WAVES) void scan_bwd_edge_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L;
    __shared__ float lds[BWD_WAVES][TILE * NP];
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, item = blockIdx.x / nblk, blk = blockIdx.x - item * nblk;
    const Lane<L, NS> w(k, k.waves, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    const bool has_z = a.z != nullptr;
    const Rows<T, L> DT(a.dt, a.dt_ld, a.cols, c, j), DY(a.dy, a.dy_ld, a.cols, c, j), Z(has_z ? a.z : a.dy, has_z ? a.z_ld : a.dy_ld, a.cols, c, j);
    const States<T, NP> C(a.C, a.c_ld, w.g, a.states, w.lane);
    float A2[NS], dhc[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn, w.full);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; dhc[i] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    int q0, q1;
    item_slots(k, item, q0, q1);
    Cursor cur(k.m);
    cur.find(q0);
    const bool begins = q0 <= cur.base, ends = cur.base + cur.tiles <= q1;
    if (ends && a.dfinal && w.ok) load_state<NS>(a.dfinal + ((int64_t)cur.s * a.cols + c) * a.states + n0, dhc, nn, w.full);
    float* Cs = lds[w.wave];
    float sd = 0.f;
    const int k0 = max(q0 - cur.base, 0), k1 = begins ? k0 : min(cur.tiles, q1 - cur.base);
    T tr[NB], gr[NB], zr[NB], cr[NP / 4];
    auto fetch = [&](int kt) {
        const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
        DT.load(row0, nr, tr); DY.load(row0, nr, gr);
        if (has_z) Z.load(row0, nr, zr);
        C.load(row0, nr, cr);
    };
    if (k0 < k1) fetch(k1 - 1);
    for (int kt = k1 - 1; kt >= k0; --kt) {
        const int nr = min(TILE, cur.end - cur.begin - kt * TILE);
        C.stage(cr, nr, Cs);
        float delta[NB], dp[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const bool ok = w.ok && b * L + j < nr;
            float slope;
            const float v = (float)tr[b] + bias, d = a.softplus ? softplus(v, slope) : v;
            delta[b] = ok ? d : 0.f;
            sd += delta[b];
            dp[b] = ok ? has_z ? (float)gr[b] * ((float)zr[b] * sigmoid<T>((float)zr[b])) : (float)gr[b] : 0.f;
        }
        if (kt > k0) fetch(kt - 1);
        wave_lds_fence();
        static_for<0, NB>([&](auto bb) {
            constexpr int b = NB - 1 - bb;
            static_for<0, L>([&](auto ii) {
                constexpr int i = L - 1 - ii;
                const float dl = from_lane<L, i>(delta[b]), dpl = from_lane<L, i>(dp[b]);
                const float* Cr = Cs + (b * L + i) * NP + n0;
#pragma unroll
                for (int e = 0; e < NS; ++e) dhc[e] = exp2_fast(dl * A2[e]) * fmaf(dpl, Cr[e], dhc[e]);
            });
        });
        wave_lds_fence();
    }
    sd = channel_sum<L>(sd);
    if (w.ok) {
        store_state<NS>(k.edge + ((int64_t)item * a.cols + c) * a.states + n0, dhc, nn, w.full);
        if (j == 0) k.sum_delta[(int64_t)item * a.cols + c] = sd;
    }
    if (blk == 0 && threadIdx.x == 0) k.cut[item] = begins || ends;
}

// Rows whose decays are worked out a second time on the way back: 4 NS registers for 4 NS exponentials of a tile, without which some would spill
template <class T> constexpr int AGAIN = sizeof(T) == 4 ? 6 : 4;
// FULL: BWD_WAVES a block, known to the compiler (8192 x 1024, 16 states: 204 us with the forward pass in place of 208); fewer where a group's channels need no more
template <class T, int L, int NS, bool FULL> __global__ __launch_bounds__(64 * BWD_WAVES, L == 16 && NS == 4 ? 1 : 2) void scan_bwd_kernel(const ScanK k) {
    constexpr int NP = L * NS, NB = TILE / L, WV = BWD_WAVES, R = RED<L, NS>;
    __shared__ float lds[WV][2][TILE * NP];
    __shared__ float red[2][WV][TILE * R];                       // two of them: one barrier a tile
    const vc_scan_args& a = k.a;
    const int nblk = a.groups * k.nblk, item = blockIdx.x / nblk, blk = blockIdx.x - item * nblk;
    const int waves = FULL ? WV : k.waves;
    const Lane<L, NS> w(k, waves, blk);
    const int c = w.c, j = w.j, n0 = w.n0, nn = w.nn;
    const bool has_z = a.z != nullptr;
    const Rows<T, L> DX(a.dx, a.dx_ld, a.cols, c, j, w.ok), DDT(a.ddt, a.ddt_ld, a.cols, c, j, w.ok), DZ(a.dz, a.dz_ld, a.cols, c, j, w.ok);
    if (item == k.items) {                                       // rows ahead of the first utterance and behind the last one
        const int head = seq_head(k.m), tail = seq_tail(k.m);
        DX.clear(0, head, c, j); DDT.clear(0, head, c, j);
        DX.clear(tail, k.m.rows, c, j); DDT.clear(tail, k.m.rows, c, j);
        if (has_z) { DZ.clear(0, head, c, j); DZ.clear(tail, k.m.rows, c, j); }
        return;
    }
    const Rows<T, L> X(a.x, a.x_ld, a.cols, c, j), DT(a.dt, a.dt_ld, a.cols, c, j), DY(a.dy, a.dy_ld, a.cols, c, j), Z(has_z ? a.z : a.dy, has_z ? a.z_ld : a.dy_ld, a.cols, c, j);
    const States<T, NP> B(a.B, a.b_ld, w.g, a.states, w.lane), C(a.C, a.c_ld, w.g, a.states, w.lane);
    float A2[NS], dA[NS], dhc[NS];
    load_state<NS>(a.A + (int64_t)c * a.states + n0, A2, nn, w.full);
#pragma unroll
    for (int i = 0; i < NS; ++i) { A2[i] *= LOG2E; dA[i] = 0.f; dhc[i] = 0.f; }
    const float Dc = a.D ? a.D[c] : 0.f, bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    int q0, q1;
    item_slots(k, item, q0, q1);
    Cursor cur(k.m);
    if (k.chunk) cur.find(q1 - 1); else cur.load(item);
    if (k.chunk && cur.base + cur.tiles > q1) carry_in<NS, false>(k, item, c, n0, nn, w.full, A2, dhc);
    float dDacc = 0.f, dbacc = 0.f;
    // waves that this block has not got add nothing (there before the first sums are taken: a barrier lies between)
    for (int o = waves * TILE * R + threadIdx.x; o < WV * TILE * R; o += 64 * waves) red[0][0][o] = red[1][0][o] = 0.f;
    float *Bs = lds[w.wave][0], *Cs = lds[w.wave][1];
    int turn = 0;
    for (int q = q1 - 1; q >= q0;) {                             // the utterances of the item, the last one first
      const int64_t hs = ((int64_t)cur.s * a.cols + c) * a.states + n0;
      const int k0 = max(q0 - cur.base, 0), k1 = min(cur.tiles, q + 1 - cur.base);
      if (cur.base + cur.tiles <= q1) {                          // its end lies in this item
#pragma unroll
        for (int i = 0; i < NS; ++i) dhc[i] = 0.f;
        if (a.dfinal && w.ok) load_state<NS>(a.dfinal + hs, dhc, nn, w.full);
      }
      T xr[NB], tr[NB], gr[NB], zr[NB], br[NP / 4], cr[NP / 4];
      float hn[NS];                                              // the state in front of the tile
      auto fetch = [&](int kt) {
        const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
        X.load(row0, nr, xr); DT.load(row0, nr, tr); DY.load(row0, nr, gr);
        if (has_z) Z.load(row0, nr, zr);
        B.load(row0, nr, br); C.load(row0, nr, cr);
        load_state<NS>(a.saved + ((int64_t)(cur.base + kt) * a.cols + c) * a.states + n0, hn, nn, w.full);
      };
      if (k0 < k1) fetch(k1 - 1);
      for (int kt = k1 - 1; kt >= k0; --kt) {
        const int row0 = cur.begin + kt * TILE, nr = min(TILE, cur.end - row0);
        float* mine = red[turn][w.wave];
        float h0[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) h0[i] = hn[i];
        B.stage(br, nr, Bs); C.stage(cr, nr, Cs);
        float xv[NB], delta[NB], slope[NB], dtx[NB], dp[NB], dzf[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const bool ok = w.ok && b * L + j < nr;
            const float g = ok ? (float)gr[b] : 0.f, v = (float)tr[b] + bias;
            xv[b] = ok ? (float)xr[b] : 0.f;
            slope[b] = 1.f;
            const float d = a.softplus ? softplus(v, slope[b]) : v;
            delta[b] = ok ? d : 0.f;
            dtx[b] = delta[b] * xv[b];
            dp[b] = g; dzf[b] = 0.f;
            if (has_z) {
                const float zv = ok ? (float)zr[b] : 0.f, sg = sigmoid<T>(zv);
                dp[b] = g * (zv * sg);
                dzf[b] = g * (sg * (1.f + zv * (1.f - sg)));
            }
        }
        wave_lds_fence();
        const auto xt = DX.tile(row0, nr), tt = DDT.tile(row0, nr), zt = DZ.tile(row0, nr);
        float av[TILE][NS], h[TILE][NS];                         // (av of the first AGAIN rows is not kept)
        Row<NS> bc[2];
        bc[0].read(Bs + n0, Cs + n0);
        static_for<0, NB>([&](auto b) {
            float acc[L];
            static_for<0, L>([&](auto i) {
                constexpr int t = b * L + i;
                if constexpr (t + 1 < TILE) bc[(t + 1) & 1].read(Bs + (t + 1) * NP + n0, Cs + (t + 1) * NP + n0);
                __builtin_amdgcn_sched_barrier(0);
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtx[b]);
                const float (&Br)[NS] = bc[t & 1].b, (&Cr)[NS] = bc[t & 1].c;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    const float hp = t ? h[t ? t - 1 : 0][e] : h0[e];
                    const float ae = exp2_fast(dl * A2[e]);
                    if constexpr (t >= AGAIN<T>) av[t][e] = ae;
                    h[t][e] = fmaf(ae, hp, dx * Br[e]);
                    sum = fmaf(Cr[e], h[t][e], sum);
                }
                acc[i] = sum;
                __builtin_amdgcn_sched_barrier(0);      // one row ahead and no more: 128 registers hold a and h
            });
            if (has_z) {
                const float yp = sums_by_row<L>(acc, j) + Dc * xv[b];
                DZ.store(zt, b, dzf[b] * yp);
            }
        });
        static_for<0, NB>([&](auto bb) {
            constexpr int b = NB - 1 - bb;
            float gacc[L], qacc[L], xb = xv[b];
            asm("" : "+v"(xb));                                  // delta x is worked out again: kept, it would cost a register for each row of a lane
            const float dtxb = delta[b] * xb;
            if (b == (NB > 1 ? NB / 2 - 1 : 0) && kt > k0) fetch(kt - 1);      // half of a and h is done with: their registers take the next tile's rows
            static_for<0, L>([&](auto ii) {
                constexpr int i = L - 1 - ii, t = b * L + i;
                if constexpr (t > 0) bc[(t - 1) & 1].read(Bs + (t - 1) * NP + n0, Cs + (t - 1) * NP + n0);
                __builtin_amdgcn_sched_barrier(0);
                const float dl = from_lane<L, i>(delta[b]), dx = from_lane<L, i>(dtxb), dpl = from_lane<L, i>(dp[b]);
                const float (&Br)[NS] = bc[t & 1].b, (&Cr)[NS] = bc[t & 1].c;
                float v[2 * NS], g = 0.f, qs = 0.f;
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    const float hp = t ? h[t ? t - 1 : 0][e] : h0[e];
                    const float dh = fmaf(dpl, Cr[e], dhc[e]);
                    v[NS + e] = dpl * h[t][e];
                    v[e] = dh * dx;
                    g = fmaf(dh, Br[e], g);
                    if constexpr (t >= AGAIN<T>) dhc[e] = av[t][e] * dh;
                    else dhc[e] = exp2_fast(dl * A2[e]) * dh;
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
            dbacc += w.ok && b * L + j < nr ? dv : 0.f;
            DX.store(xt, b, fmaf(delta[b], g, dp[b] * Dc));
            DDT.store(tt, b, dv);
        });
        __syncthreads();
        for (int o = threadIdx.x; o < nr * 2 * NP; o += 64 * waves) {
            const int t = o / (2 * NP), e = o % (2 * NP), n = e % NP, it = (e / NP) * NS + n % NS;
            const float* at = red[turn][0] + t * R + item_at<L, NS>(it, n / NS);
            float f[WV * SPLIT<L, NS>];
#pragma unroll
            for (int v = 0; v < WV; ++v)
#pragma unroll
                for (int u = 0; u < SPLIT<L, NS>; ++u) f[v * SPLIT<L, NS> + u] = at[v * TILE * R + 4 * u];
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < WV * SPLIT<L, NS>; ++v) sum += f[v];
            k.part[((int64_t)blk * k.m.rows + row0 + t) * (2 * NP) + e] = sum;
        }
        turn ^= 1;
      }
      if (cur.base >= q0 && cur.base < q1 && a.dinitial && w.ok) store_state<NS>(a.dinitial + hs, dhc, nn, w.full);       // its beginning lies in this item
      if (cur.base <= q0 || cur.s == 0) break;
      q = min(cur.base, q) - 1;
      cur.load(cur.s - 1);
    }
    if (w.ok) store_state<NS>(k.dapart + ((int64_t)item * a.cols + c) * a.states + n0, dA, nn, w.full);
    const float d = channel_sum<L>(dDacc), b = channel_sum<L>(dbacc);
    if (w.ok && j == 0) {
        k.chpart[((int64_t)item * 2) * a.cols + c] = d;
        k.chpart[((int64_t)item * 2 + 1) * a.cols + c] = b;
    }
}

// What the main pass left in parts: dB and dC are summed over the blocks of a group and rounded once (blocks [0, bc)), dA, dD and ddt_bias over the items
// (16 columns of sums a block, 16 threads a column).  64 x 128 x 1024: 6 us.
template <class T> __global__ __launch_bounds__(256) void scan_finish_kernel(const ScanK k, int np, int bc) {
    __shared__ float red[16][17];
    const vc_scan_args& a = k.a;
    if ((int)blockIdx.x < bc) {
        const int64_t w = (int64_t)2 * np * a.groups;
        const int head = seq_head(k.m), tail = seq_tail(k.m);
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)k.m.rows * w; i += (int64_t)bc * 256) {
            const int64_t r = i / w;
            const int e = (int)(i - r * w), g = e / (2 * np), m = e % (2 * np), n = m % np;
            if (n >= a.states) continue;
            T* dst = m < np ? (T*)a.dB + r * a.db_ld : (T*)a.dC + r * a.dc_ld;
            dst += g * a.states + n;
            if (r < head || r >= tail) { if (a.zero_tail) *dst = (T)0.f; continue; }
            float s = 0.f;
#pragma unroll 8
            for (int b = 0; b < k.nblk; ++b) s += k.part[((int64_t)(g * k.nblk + b) * k.m.rows + r) * (2 * np) + m];
            *dst = (T)s;
        }
        return;
    }
    // dapart [items][cols * states], chpart [items][2 * cols]
    const int64_t na = (int64_t)a.cols * a.states, i = (int64_t)(blockIdx.x - bc) * 16 + (threadIdx.x & 15);
    const bool second = i >= na;
    const int64_t e = second ? i - na : i, width = second ? 2 * (int64_t)a.cols : na;
    const float* src = second ? k.chpart : k.dapart;
    const int w = threadIdx.x >> 4;
    float s = 0.f;
    if (e < width) {
        int q = w;
        for (; q + 112 < k.items; q += 128) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = src[(q + 16 * u) * width + e];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
#pragma unroll 4
        for (; q < k.items; q += 16) s += src[q * width + e];
    }
    red[w][threadIdx.x & 15] = s;
    __syncthreads();
    if (w || e >= width) return;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < 16; ++u) s += red[u][threadIdx.x];
    if (!second) a.dA[e] = s;
    else if (e < a.cols) { if (a.dD) a.dD[e] = s; }
    else if (a.ddt_bias) a.ddt_bias[e - a.cols] = s;
}

constexpr double BWD_MARGIN = 4;
constexpr int64_t BWD_RUN_WAVES = 2048;                          // two waves a SIMD is what its registers allow
static int bwd_setup(const char* who, const vc_scan_args* a, ScanK* k, int64_t* floats) {
    VC_ARG(a, "%s: null pointer", who);
    VC_CHECK(scan_setup(who, a, BWD_WAVES, BWD_RUN_WAVES, BWD_MARGIN, k));
    const int64_t part = (int64_t)a->groups * k->nblk * a->rows * 2 * scan_padded(a->states);
    const int64_t da = (int64_t)k->items * a->cols * a->states, ch = (int64_t)k->items * 2 * a->cols;
    *floats = part + da + ch + scan_edge_floats(*k);
    k->part = a->work; k->dapart = a->work + part; k->chpart = k->dapart + da;
    scan_edge_place(k, k->chpart + ch);
    return 0;
}
extern "C" int64_t vc_selective_scan_bwd_work(const vc_scan_args* a) {
    ScanK k; int64_t n;
    return bwd_setup("vc_selective_scan_bwd_work", a, &k, &n) ? VC_E_ARG : n;
}
template <class T, int L, int NS> static int scan_bwd_l(const ScanK& k, hipStream_t s) {
    const int64_t blocks = (int64_t)k.a.groups * k.nblk * (k.items + (k.a.zero_tail && k.m.off ? 1 : 0));
    const int64_t bc = std::min<int64_t>(((int64_t)k.m.rows * 2 * L * NS * k.a.groups + 255) / 256, 1 << 22);
    const int64_t eb = (int64_t)k.a.groups * k.nblk * k.items;
    VC_ARG(blocks < (1LL << 31) && eb < (1LL << 31), "vc_selective_scan_bwd: too many utterances and channels for one launch");
    if (k.chunk) {
        hipLaunchKernelGGL((scan_bwd_edge_kernel<T, L, NS>), dim3((unsigned)eb), dim3(64 * k.waves), 0, s, k);
        VC_CHECK(scan_carry(k, false, s));
    }
    if (k.waves == BWD_WAVES) hipLaunchKernelGGL((scan_bwd_kernel<T, L, NS, true>), dim3((unsigned)blocks), dim3(64 * BWD_WAVES), 0, s, k);
    else hipLaunchKernelGGL((scan_bwd_kernel<T, L, NS, false>), dim3((unsigned)blocks), dim3(64 * k.waves), 0, s, k);
    const int64_t pc = ((int64_t)k.a.cols * (k.a.states + 2) + 15) / 16;
    VC_ARG(bc + pc < (1LL << 31), "vc_selective_scan_bwd: too many rows and channels for one launch");
    hipLaunchKernelGGL((scan_finish_kernel<T>), dim3((unsigned)(bc + pc)), dim3(256), 0, s, k, L * NS, (int)bc);
    VC_HIP(hipGetLastError());
    return 0;
}
template <class T> static int scan_bwd_t(const ScanK& k, hipStream_t s) { return SCAN_LAYOUT(T, k.a.states, scan_bwd_l, k, s); }
extern "C" int vc_selective_scan_bwd(const vc_scan_args* a, void* stream) {
    ScanK k; int64_t need;
    VC_CHECK(bwd_setup("vc_selective_scan_bwd", a, &k, &need));
    VC_ARG(a->A && a->dA && (a->rows == 0 || (a->x && a->dt && a->B && a->C && a->dy && a->dx && a->ddt && a->dB && a->dC && a->saved)), "vc_selective_scan_bwd: null pointer");
    VC_ARG(!a->z || a->dz || a->rows == 0, "vc_selective_scan_bwd: z has a gradient, dz is null");
    VC_ARG(!a->dinitial || a->dinitial != a->dfinal, "vc_selective_scan_bwd: dinitial may not be dfinal: not in place, an utterance's beginning and end may lie in two runs");
    if (!a->z) k.a.dz = nullptr;
    if (a->saved_floats < vc_selective_scan_saved(a) && a->rows) { vc_set_error("vc_selective_scan_bwd: saved is too small"); return VC_E_NOMEM; }
    if (a->work_floats < need || !a->work) { vc_set_error("vc_selective_scan_bwd: work is too small (%lld floats needed)", (long long)need); return VC_E_NOMEM; }
    return SEQ_TYPES(a->type, scan_bwd_t, k, (hipStream_t)stream);
}
