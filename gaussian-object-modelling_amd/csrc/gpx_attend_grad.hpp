// gpx_attend_grad.hpp -- the kernels of gpx_attend_backward.
//
// With p_ij = exp(s_ij - lse_i) and D_i = <dO_i, O_i>:  dV_j = sum_i p_ij dO_i,  dS_ij = p_ij (<dO_i, V_j> - D_i),
// dQ_i = scale sum_j dS_ij K_j,  dK_j = scale sum_i dS_ij Q_i; for shared heads the sums over i run over the whole group, which
// the packed rows do by themselves.  Two kernels, each forming p and dS again for its own sums (7 products instead of 5): dQ
// with the rows held by the wave, dK and dV with the keys held by the wave.  No atomics: every sum has a fixed order.
#pragma once
#include "gpx_attend_tile.hpp"

namespace gpx {
namespace attend {

// lse in log2 units (+inf where a row has no weights, so that every p is 0) and <dO, O>, one lane group of 16 per row
template <typename T>
__global__ __launch_bounds__(256) void attend_stat_kernel(AttendBwd a, long rows)
{
    const AttendRows &rw = a.rows;
    const int sub = threadIdx.x & 15, H = rw.Hk * rw.G;
    const long rid = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool on = rid < rows;
    const int i = on ? (int)(rid % rw.M) : 0;
    const long bh = on ? rid / rw.M : 0;
    const int h = (int)(bh % H);
    const long b = bh / H;
    float s = 0.0f;
    const bool valid = on && (!rw.len || i < rw.len[b]);
    const int d = 8 * sub;
    if (valid && d < rw.D) {
        const x8<T> g = *reinterpret_cast<const x8<T> *>((const T *)a.dout + b * a.gb + i * a.gr + h * a.gh + d);
        const x8<T> o = *reinterpret_cast<const x8<T> *>((const T *)a.o + b * a.ob + i * a.orow + h * a.oh + d);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            s += (float)g[j] * (float)o[j];
    }
#pragma unroll
    for (int k = 8; k; k >>= 1)
        s += __shfl_xor(s, k);
    if (on && sub == 0) {
        const float lse = valid ? a.lse[rid] : NEG_INF;
        const bool none = lse == NEG_INF;
        a.stat[rid] = make_float2(none ? POS_INF : lse * 1.44269504088896f, none ? 0.0f : s);
    }
}

// dQ: waves as in the forward kernel.  S^T = K Q^T and dP^T = V dO^T, then dQ^T += K^T dS^T.
template <typename T, int DT, int WM>
struct DqShape {
    static constexpr int WK = 4 / WM;
    static constexpr int KT = 32;
    static constexpr int BN = KT * WK;
    static constexpr int BM = 32 * WM;
};

template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && (WM == 4 || DT <= 2) ? 2 : 1)) void attend_dq_kernel(AttendBwd a)
{
    using TL = Tile<T, DT>;
    using SH = DqShape<T, DT, WM>;
    constexpr int BN = SH::BN, WK = SH::WK, KT = SH::KT;
    __shared__ __attribute__((aligned(16))) char lds[2 * BN * TL::ROWB < 512 ? 512 : 2 * BN * TL::ROWB];
    char *kt = lds, *vt = lds + BN * TL::ROWB;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;
    const AttendRows &rw = a.rows;
    const int mtiles = (rw.R + SH::BM - 1) / SH::BM;
    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    const int mt = id % mtiles;
    id /= mtiles;
    const int split = id % a.q_splits;
    id /= a.q_splits;
    const int hk = id % rw.Hk, bz = id / rw.Hk;

    const RowAt at = row_at(rw, bz, hk, mt * SH::BM + wm * 32 + (lane & 31));
    const int len = clamped(a.keys.len, bz, a.keys.n);
    const int begin = split * a.q_chunk, end = min(len, begin + a.q_chunk);

    x8<T> qf[2 * DT], gf[2 * DT];
    load_row_frags<T, DT>(qf, (const T *)rw.q + (at.valid ? at.b * rw.qb + at.i * rw.qr + at.h * rw.qh : 0), at.valid, rw.D, lane);
    load_row_frags<T, DT>(gf, (const T *)a.dout + (at.valid ? at.b * a.gb + at.i * a.gr + at.h * a.gh : 0), at.valid, rw.D, lane);
    float2 stat = make_float2(POS_INF, 0.0f);
    if (at.valid)
        stat = a.stat[((long)at.b * rw.Hk * rw.G + at.h) * rw.M + at.i];

    f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            dq[d][i] = 0.0f;

    const T *kp = (const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh;
    const T *vp = (const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh;
    const unsigned char *mask = a.keys.mask ? a.keys.mask + bz * a.keys.mask_b : nullptr;
    const auto counts = [mask](int j) { return !mask || mask[j]; };
    const int rbase = TL::row_base(lane), cbase = TL::col_base(lane);

    Stage<T, DT, BN, 256> sk, sv;
    if (begin < end) {
        sk.load(kp, a.keys.kr, begin, end, rw.D, tid, counts);
        sv.load(vp, a.keys.vr, begin, end, rw.D, tid, counts);
    }
    for (int n0 = begin; n0 < end; n0 += BN) {
        const int j = n0 + wk * KT + (lane & 31);
        const unsigned seen = (unsigned)__ballot(j < end && counts(j));
        __syncthreads();
        sk.store(kt, tid);
        sv.store(vt, tid);
        __syncthreads();
        if (n0 + BN < end) {
            sk.load(kp, a.keys.kr, n0 + BN, end, rw.D, tid, counts);
            sv.load(vp, a.keys.vr, n0 + BN, end, rw.D, tid, counts);
        }
        if (seen == 0)
            continue;
        f32x16 sc, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[i] = dp[i] = 0.0f;
#pragma unroll
        for (int t = 0; t < TL::KS; ++t) {
            sc = mma(TL::row_frag(kt, rbase, wk * KT, t), qf[t], sc);
            dp = mma(TL::row_frag(vt, rbase, wk * KT, t), gf[t], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[i] = exp2_(sc[i] * a.c - stat.x) * (dp[i] - stat.y);
        if (seen != 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[i] = bit_of(seen, half, i) ? sc[i] : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const x8<T> ds = as_operand<T>(sc, t);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                dq[d] = mma(TL::col_frag(kt, cbase, wk * KT + 16 * t, d), ds, dq[d]);
        }
    }
    if constexpr (WK > 1) {
        constexpr int PIECE = 64 * 16 * DT;
        static_assert((WK - 1) * WM * PIECE * 4 <= 2 * BN * TL::ROWB, "the join uses the tiles' memory");
        float *pc = reinterpret_cast<float *>(lds);
        __syncthreads();
        if (wk > 0) {
            float *w = pc + ((wk - 1) * WM + wm) * PIECE;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    w[(d * 16 + i) * 64 + lane] = dq[d][i];
        }
        __syncthreads();
        if (wk > 0)
            return;
#pragma unroll
        for (int k = 1; k < WK; ++k) {
            const float *w = pc + ((k - 1) * WM + wm) * PIECE;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    dq[d][i] += w[(d * 16 + i) * 64 + lane];
        }
    }
    if (!at.exists)
        return;
    if (a.pq) {
        const long rid = ((long)at.b * rw.M + at.i) * ((long)rw.Hk * rw.G) + at.h;
        float *p = a.pq + ((long)split * ((long)rw.grid_b * rw.M * rw.Hk * rw.G) + rid) * rw.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int f = 32 * d + 8 * x + 4 * half;
                if (f < rw.D)
                    *reinterpret_cast<f32x4 *>(p + f) = f32x4{dq[d][4 * x], dq[d][4 * x + 1], dq[d][4 * x + 2], dq[d][4 * x + 3]};
            }
        return;
    }
    T *p = (T *)a.dq + at.b * a.dqb + at.i * a.dqr + at.h * a.dqh;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int f = 32 * d + 8 * x + 4 * half;
            x4<T> w;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = (T)(dq[d][4 * x + k] * a.scale);
            if (f < rw.D)
                *reinterpret_cast<x4<T> *>(p + f) = w;
        }
}

// dK, dV: 4 waves of 32 keys each; the rows pass through LDS in tiles of BR.  S = Q K^T and dP = dO V^T with a lane holding one
// key, then dV^T += dO^T P and dK^T += Q^T dS.
template <typename T, int DT>
__global__ __launch_bounds__(256, 1) void attend_dkv_kernel(AttendBwd a)
{
    using TL = Tile<T, DT>;
    constexpr int BR = sizeof(T) == 2 ? 64 : 32;
    __shared__ __attribute__((aligned(16))) char lds[2 * BR * TL::ROWB];
    __shared__ __attribute__((aligned(16))) float st_lse[BR];
    __shared__ __attribute__((aligned(16))) float st_d[BR];
    char *qt = lds, *gt = lds + BR * TL::ROWB;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const AttendRows &rw = a.rows;
    const int ktiles = (a.keys.n + ATTEND_DKV_KEYS - 1) / ATTEND_DKV_KEYS;
    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    const int ktile = id % ktiles;
    id /= ktiles;
    const int split = id % a.k_splits;
    id /= a.k_splits;
    const int hk = id % rw.Hk, bz = id / rw.Hk;

    const int len = clamped(a.keys.len, bz, a.keys.n);
    const int key = ktile * ATTEND_DKV_KEYS + wave * 32 + (lane & 31);
    const bool exists = key < a.keys.n;
    const bool counts = key < len && (!a.keys.mask || a.keys.mask[bz * a.keys.mask_b + key]);
    const int begin = split * a.k_chunk, end = min(rw.R, begin + a.k_chunk);

    x8<T> kf[2 * DT], vf[2 * DT];
    load_row_frags<T, DT>(kf, (const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh + (counts ? key * a.keys.kr : 0), counts, rw.D, lane);
    load_row_frags<T, DT>(vf, (const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh + (counts ? key * a.keys.vr : 0), counts, rw.D, lane);

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            dk[d][i] = dv[d][i] = 0.0f;

    const int rbase = TL::row_base(lane), cbase = TL::col_base(lane);
    constexpr int N = (BR * TL::NCH + 255) / 256;
    u32x4 rq[N], rg[N];
    float2 rs;
    const auto load = [&](int r0) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int cid = tid + x * 256, row = cid / TL::NCH, c = cid - row * TL::NCH;
            u32x4 zq = {0, 0, 0, 0}, zg = {0, 0, 0, 0};
            if ((BR * TL::NCH % 256 == 0 || row < BR) && r0 + row < end && c * TL::EPC < rw.D) {
                const RowAt w = row_at(rw, bz, hk, r0 + row);
                if (w.valid) {
                    zq = *reinterpret_cast<const u32x4 *>((const T *)rw.q + w.b * rw.qb + w.i * rw.qr + w.h * rw.qh + c * TL::EPC);
                    zg = *reinterpret_cast<const u32x4 *>((const T *)a.dout + w.b * a.gb + w.i * a.gr + w.h * a.gh + c * TL::EPC);
                }
            }
            rq[x] = zq;
            rg[x] = zg;
        }
        rs = make_float2(POS_INF, 0.0f);
        if (tid < BR && r0 + tid < end) {
            const RowAt w = row_at(rw, bz, hk, r0 + tid);
            if (w.valid)
                rs = a.stat[((long)w.b * rw.Hk * rw.G + w.h) * rw.M + w.i];
        }
    };
    const bool work = ktile * ATTEND_DKV_KEYS < len;  // else nothing here counts: zeros
    if (work && begin < end)
        load(begin);
    for (int r0 = begin; work && r0 < end; r0 += BR) {
        __syncthreads();
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int cid = tid + x * 256, row = cid / TL::NCH, c = cid - row * TL::NCH;
            if (BR * TL::NCH % 256 == 0 || row < BR) {
                *reinterpret_cast<u32x4 *>(qt + TL::place(row, c)) = rq[x];
                *reinterpret_cast<u32x4 *>(gt + TL::place(row, c)) = rg[x];
            }
        }
        if (tid < BR) {
            st_lse[tid] = rs.x;
            st_d[tid] = rs.y;
        }
        __syncthreads();
        if (r0 + BR < end)
            load(r0 + BR);
#pragma unroll
        for (int s = 0; s < BR / 32; ++s) {
            f32x16 p, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                p[i] = dp[i] = 0.0f;
#pragma unroll
            for (int t = 0; t < TL::KS; ++t) {
                p = mma(TL::row_frag(qt, rbase, 32 * s, t), kf[t], p);
                dp = mma(TL::row_frag(gt, rbase, 32 * s, t), vf[t], dp);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 ls = *reinterpret_cast<const f32x4 *>(st_lse + 32 * s + 8 * x + 4 * half);
                const f32x4 ds = *reinterpret_cast<const f32x4 *>(st_d + 32 * s + 8 * x + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 4 * x + j;
                    p[i] = exp2_(p[i] * a.c - ls[j]);
                    dp[i] = p[i] * (dp[i] - ds[j]);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const x8<T> w = as_operand<T>(p, t), ws = as_operand<T>(dp, t);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    dv[d] = mma(TL::col_frag(gt, cbase, 32 * s + 16 * t, d), w, dv[d]);
                    dk[d] = mma(TL::col_frag(qt, cbase, 32 * s + 16 * t, d), ws, dk[d]);
                }
            }
        }
    }
    if (!exists)
        return;
    // a key that does not count had zeros for its fragments: its sums are of finite weights but not zero
    const float fk = counts ? 1.0f : 0.0f;
    if (a.pk) {
        const long at = ((long)split * rw.grid_b * rw.Hk + (long)bz * rw.Hk + hk) * a.keys.n + key;
        float *pk = a.pk + at * rw.D, *pv = a.pv + at * rw.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int f = 32 * d + 8 * x + 4 * half;
                f32x4 wk, wv;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    wk[j] = fk == 0.0f ? 0.0f : dk[d][4 * x + j];
                    wv[j] = fk == 0.0f ? 0.0f : dv[d][4 * x + j];
                }
                if (f < rw.D) {
                    *reinterpret_cast<f32x4 *>(pk + f) = wk;
                    *reinterpret_cast<f32x4 *>(pv + f) = wv;
                }
            }
        return;
    }
    T *pk = (T *)a.dk + bz * a.dkb + key * a.dkr + hk * a.dkh, *pv = (T *)a.dv + bz * a.dvb + key * a.dvr + hk * a.dvh;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int f = 32 * d + 8 * x + 4 * half;
            x4<T> wk, wv;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                wk[j] = fk == 0.0f ? (T)0.0f : (T)(dk[d][4 * x + j] * a.scale);
                wv[j] = fk == 0.0f ? (T)0.0f : (T)dv[d][4 * x + j];
            }
            if (f < rw.D) {
                *reinterpret_cast<x4<T> *>(pk + f) = wk;
                *reinterpret_cast<x4<T> *>(pv + f) = wv;
            }
        }
}

// out[row] = f sum_s p[s][row], in slot order; rows of D values, four per lane.  Row -> (batch, n, head) by the strides.
struct AttendSum {
    const float *p;
    int slots, D, n, H;  // row = (b n + i) H + h  or, head_first, (b H + h) n + i
    long rows;
    int head_first;
    float f;
    void *out;
    long ob, orow, oh;
};
template <typename T>
__global__ __launch_bounds__(256) void attend_sum_kernel(AttendSum a)
{
    const int q = a.D >> 2;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.rows * q)
        return;
    const long row = id / q;
    const int d = 4 * (int)(id - row * q);
    f32x4 s = {0, 0, 0, 0};
    for (int k = 0; k < a.slots; ++k)
        s += *reinterpret_cast<const f32x4 *>(a.p + ((long)k * a.rows + row) * a.D + d);
    long b, i, h;
    if (a.head_first) {
        i = row % a.n;
        h = row / a.n % a.H;
        b = row / a.n / a.H;
    } else {
        h = row % a.H;
        i = row / a.H % a.n;
        b = row / a.H / a.n;
    }
    x4<T> w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w[j] = (T)(s[j] * a.f);
    *reinterpret_cast<x4<T> *>((T *)a.out + b * a.ob + i * a.orow + h * a.oh + d) = w;
}

template <typename T, int DT, int WM>
void launch_dq_shape(const AttendBwd &a, hipStream_t st)
{
    const int mtiles = (a.rows.R + 32 * WM - 1) / (32 * WM);
    const unsigned grid = (unsigned)((long)mtiles * a.q_splits * a.rows.Hk * a.rows.grid_b);
    hipLaunchKernelGGL((attend_dq_kernel<T, DT, WM>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T, int DT>
void launch_bwd_dim(const AttendBwd &a, hipStream_t st)
{
    if (a.rows.R > 0 && a.rows.M > 0) {
        switch (attend_block_rows(sizeof(T) == 4, a.rows.D, a.rows.R)) {
        case 32:
        if constexpr (sizeof(T) == 2 || DT <= 2)
            launch_dq_shape<T, DT, 1>(a, st);
        break;
        case 64: launch_dq_shape<T, DT, 2>(a, st); break;
        default: launch_dq_shape<T, DT, 4>(a, st); break;
        }
    }
    const int ktiles = (a.keys.n + ATTEND_DKV_KEYS - 1) / ATTEND_DKV_KEYS;
    const unsigned grid = (unsigned)((long)ktiles * a.k_splits * a.rows.Hk * a.rows.grid_b);
    if (grid)
        hipLaunchKernelGGL((attend_dkv_kernel<T, DT>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T>
void launch_sum(const AttendSum &s, hipStream_t st)
{
    const long lanes = s.rows * (s.D / 4);
    if (lanes)
        hipLaunchKernelGGL((attend_sum_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st, s);
}

}  // namespace attend

template <typename T>
void attend_launch_bwd(const AttendBwd &a, hipStream_t st)
{
    const AttendRows &rw = a.rows;
    const int H = rw.Hk * rw.G;
    const long rows = (long)rw.grid_b * rw.M * H;
    if (rows)
        hipLaunchKernelGGL((attend::attend_stat_kernel<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a, rows);
    switch ((rw.D + 31) / 32) {
    case 1: attend::launch_bwd_dim<T, 1>(a, st); break;
    case 2: attend::launch_bwd_dim<T, 2>(a, st); break;
    case 3: attend::launch_bwd_dim<T, 3>(a, st); break;
    default: attend::launch_bwd_dim<T, 4>(a, st); break;
    }
    if (a.pq)
        attend::launch_sum<T>({a.pq, a.q_splits, rw.D, rw.M, H, rows, 0, a.scale, a.dq, a.dqb, a.dqr, a.dqh}, st);
    if (a.pk) {
        const long kr = (long)rw.grid_b * rw.Hk * a.keys.n;
        attend::launch_sum<T>({a.pk, a.k_splits, rw.D, a.keys.n, rw.Hk, kr, 1, a.scale, a.dk, a.dkb, a.dkr, a.dkh}, st);
        attend::launch_sum<T>({a.pv, a.k_splits, rw.D, a.keys.n, rw.Hk, kr, 1, 1.0f, a.dv, a.dvb, a.dvr, a.dvh}, st);
    }
}

}  // namespace gpx
