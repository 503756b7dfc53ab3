// gpx_attend_grad.hpp -- the kernels of gpx_attend_backward.
//
// With p_ij = exp(s_ij - lse_i) and D_i = <dO_i, O_i>:  dV_j = sum_i p_ij dO_i,  dS_ij = p_ij (<dO_i, V_j> - D_i),
// dQ_i = scale sum_j dS_ij K_j,  dK_j = scale sum_i dS_ij Q_i; for shared heads the sums over i run over the whole group, which
// the packed rows do by themselves.  Two kernels, each forming p and dS again for its own sums (7 products instead of 5): dQ
// with the rows held by the wave, dK and dV with the keys held by the wave.  No atomics: every sum has a fixed order.  (One kernel
// with 5 products would have to add dQ up over the key tiles: in memory, 64 partial sums of it at 8191 keys, or by atomics, whose
// order changes the result.)
// bf16, 2 x 4096 queries, 8191 keys, 16 heads of 128, from card to card: dQ 736 to 752 us = 1120 to 1096 TFLOP/s, dK dV 1010 to 1061 us =
// 1088 to 1036 TFLOP/s -- about the rate of the library's large products; the 7 products are what is left.  Ragged and small shapes
// are bound by latency: eight objects with 16 / 4 heads of 64 in fp16: 47 and 63 us (without the powers of two below: 42 and 60).
#pragma once
#include <type_traits>

#include "gpx_attend_tile.hpp"

namespace gpx {
namespace attend {

// fp16 has normal numbers from 2^-14 to 2^15 only, and dS = p (dP - D) may lie anywhere: p as small as 1 / keys, dO of any size (loss
// scaling).  Each row (dQ) or entry (dK) carries a power of two f: f dS is what is rounded and summed, 1 / f goes over the
// sum at the end.  f starts far too large and only falls: where the largest |f dS| of a tile passes 2^15 it is brought to 2^7 .. 2^8,
// what is summed so far with it, and 2^8 of growth are left.  So a dS down to 2^-21 of its row's (entry's) largest so far has all
// its bits, and none overflows.  The weights for dV are at most 1 and are rounded as 2^12 p.
// bf16 and fp32 (pieces of bf16) have fp32's range and take dS as it is.
template <typename T> constexpr bool NARROW = std::is_same_v<T, _Float16>;
template <typename T> constexpr float P_LIFT = NARROW<T> ? 12.0f : 0.0f;  // (0x1p-12f at the end)
constexpr float F_START = 0x1p60f, F_MOST = 0x1p15f;
// the factor that brings top, where it is above F_MOST, to 2^7 .. 2^8
__device__ __forceinline__ float bring_down(float top)
{
    return top > F_MOST ? fminf(__builtin_amdgcn_ldexpf(1.0f, 8 - __builtin_amdgcn_frexp_expf(top)), 1.0f) : 1.0f;  // (infinities: 1)
}
__device__ __forceinline__ float reciprocal_of_power(float f) { return __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(unsigned, f)); }
__device__ __forceinline__ float largest(const f32x16 &w)
{
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        top = fmaxf(top, __builtin_fabsf(w[i]));
    return max_both_halves(top);
}
template <int DT>
__device__ __forceinline__ void times(f32x16 (&acc)[DT], float g)
{
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            acc[d][i] *= g;
}

// dQ: waves and tiles as in the forward kernel.  S^T = K Q^T and dP^T = V dO^T, then dQ^T += K^T dS^T.
// The first piece of the key range also leaves each row's statistics for the dK, dV kernel, where that runs behind this one.
template <typename T, int DT, int WM>
__device__ __forceinline__ void attend_dq_block(const AttendBwd &a, char *lds, float *bias, unsigned id, unsigned total)
{
    using TL = Tile<T, DT>;
    constexpr int WK = 4 / WM, KT = 32, BN = attend_dq_bn(WM);
    using FL = Fill<T, DT, BN>;
    constexpr int TILE_B = BN * TL::ROWB;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;
    const AttendRows &rw = a.rows;
    int mt, u;
    place_block(id, total, a.q_order, a.mtiles, a.by_mtiles, mt, u);
    const int us = rw.by_hk(u), hk = u - us * rw.Hk;
    const int turn = a.by_q_splits(us), split = us - turn * a.q_splits;
    const int bz = nth_longest(a.keys, rw.grid_b, turn);

    const RowAt at = row_at(rw, bz, hk, mt * 32 * WM + wm * 32 + (lane & 31));
    const int len = clamped(a.keys.len, bz, a.keys.n);
    const int begin = split * a.q_chunk, end = min(len, begin + a.q_chunk);

    const unsigned ksb = (unsigned)(a.keys.kr * sizeof(T)), vsb = (unsigned)(a.keys.vr * sizeof(T));
    const char *kp = (const char *)((const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh);
    const char *vp = (const char *)((const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh);
    const unsigned char *mask = a.keys.mask ? a.keys.mask + bz * a.keys.mask_b : nullptr;
    const unsigned lds0 = lds_offset(lds);

    unsigned ko[FL::N], vo[FL::N];
#pragma unroll
    for (int x = 0; x < FL::N; ++x) {
        const unsigned c = FL::chunk(x, wave, lane, rw.D), r = FL::row(x, wave, lane);
        ko[x] = c == DMA_OUT ? DMA_OUT : r * ksb + c;
        vo[x] = c == DMA_OUT ? DMA_OUT : r * vsb + c;
    }
    unsigned mb[FL::N + 1];
    const auto look = [&](int n0) {
        if (!mask)
            return;
#pragma unroll
        for (int x = 0; x < FL::N; ++x) {
            const int j = n0 + FL::row(x, wave, lane);
            mb[x] = j < end ? mask[j] : 0;
        }
        const int j = n0 + tid;
        mb[FL::N] = tid < BN && j < end ? mask[j] : 0;
    };
    const auto fetch = [&](int n0, int stage) {
        const unsigned left = (unsigned)(end - n0);
        const u32x4 kd = dma_buffer(kp + (long)n0 * ksb, (unsigned)min((unsigned long long)left * ksb, (unsigned long long)DMA_MOST));
        const u32x4 vd = dma_buffer(vp + (long)n0 * vsb, (unsigned)min((unsigned long long)left * vsb, (unsigned long long)DMA_MOST));
        const unsigned at0 = lds0 + stage * 2 * TILE_B;
        if (mask) {
#pragma unroll
            for (int x = 0; x < FL::N; ++x)
                if (FL::on(x, wave)) {
                    dma16(kd, mb[x] ? ko[x] : DMA_OUT, at0 + FL::lds(x, wave));
                    dma16(vd, mb[x] ? vo[x] : DMA_OUT, at0 + TILE_B + FL::lds(x, wave));
                }
        } else {
#pragma unroll
            for (int x = 0; x < FL::N; ++x)
                if (FL::on(x, wave)) {
                    dma16(kd, ko[x], at0 + FL::lds(x, wave));
                    dma16(vd, vo[x], at0 + TILE_B + FL::lds(x, wave));
                }
        }
        if ((mask || n0 + BN > end) && tid < BN)
            bias[stage * BN + tid] = n0 + tid < end && (!mask || mb[FL::N]) ? 0.0f : NEG_INF;
    };
    if (begin < end) {
        look(begin);
        fetch(begin, 0);
        look(begin + BN);
    }

    Frag<T> qf[2 * DT], gf[2 * DT];
    load_row_frags<T, DT>(qf, (const T *)rw.q + (at.valid ? at.b * rw.qb + at.i * rw.qr + at.h * rw.qh : 0), at.valid, rw.D, lane);
    load_row_frags<T, DT>(gf, (const T *)a.dout + (at.valid ? at.b * a.gb + at.i * a.gr + at.h * a.gh : 0), at.valid, rw.D, lane);
    // lse in log2 units (+inf where the row has no weights, so that every p is 0), and <dO, O>
    float lse = POS_INF, dd = 0.0f;
    bool weights;  // the row has some: else its gradient is zero, whatever it holds and whatever the entries hold
    {
        Frag<T> of[2 * DT];
        load_row_frags<T, DT>(of, (const T *)a.o + (at.valid ? at.b * a.ob + at.i * a.orow + at.h * a.oh : 0), at.valid, rw.D, lane);
        const long rid = ((long)at.b * rw.Hk * rw.G + at.h) * rw.M + at.i;
        const float from = at.valid ? a.lse[rid] : NEG_INF;
#pragma unroll
        for (int t = 0; t < 2 * DT; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                dd += gf[t][j] * of[t][j];
        dd = sum_both_halves(dd);
        weights = from != NEG_INF;
        if (weights)
            lse = from * 1.44269504088896f;
        else
            dd = 0.0f;
        if (!a.fused && split == 0 && wk == 0 && half == 0 && at.exists) {
            a.stat[rid] = lse - P_LIFT<T>;
            a.stat[(long)rw.grid_b * rw.Hk * rw.G * rw.M + rid] = dd;
        }
    }

    f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            dq[d][i] = 0.0f;
    float f = F_START, fdd = dd * F_START;  // (NARROW)

    const auto step = [&](int stage, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        const char *kt = lds, *vt = lds + TILE_B;
        const int rbase = TL::row_base(lane) + stage * 2 * TILE_B, cbase = TL::col_base(lane) + stage * 2 * TILE_B;
        f32x16 sc, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[i] = dp[i] = 0.0f;
        if constexpr (EDGE) {  // -inf where the key does not count: its weight, and with it dS, is zero
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 w = *reinterpret_cast<const f32x4 *>(&bias[stage * BN + wk * KT + 8 * x + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sc[4 * x + j] = w[j];
            }
        }
#pragma unroll
        for (int t = 0; t < TL::KS; ++t) {
            sc = mma(TL::row_frag(kt, rbase, wk * KT, t), qf[t], sc);
            dp = mma(TL::row_frag(vt, rbase, wk * KT, t), gf[t], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[i] = exp2_(sc[i] * a.c - lse) * (NARROW<T> ? dp[i] * f - fdd : dp[i] - dd);
        if constexpr (NARROW<T>) {
            const float top = largest(sc);
            if (__any(top > F_MOST)) {
                const float g = bring_down(top);
                f *= g;
                fdd *= g;
                times<DT>(dq, g);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[i] *= g;
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Frag<T> ds = as_operand<T>(sc, t);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                dq[d] = mma(TL::col_frag(kt, cbase, wk * KT + 16 * t, d), ds, dq[d]);
        }
    };
    const int plain = mask || end < begin ? begin : begin + (end - begin) / BN * BN;
    int stage = 0;
    const auto steps = [&](int from, int to, auto edge) {
        for (int n0 = from; n0 < to; n0 += BN, stage ^= 1) {
            dma_wait();
            __syncthreads();
            if (n0 + BN < end) {
                fetch(n0 + BN, stage ^ 1);
                look(n0 + 2 * BN);
            }
            step(stage, edge);
        }
    };
    steps(begin, plain, std::false_type());
    steps(plain, end, std::true_type());
    if constexpr (NARROW<T>)
        times<DT>(dq, reciprocal_of_power(f));
    if constexpr (WK > 1) {
        constexpr int PIECE = 64 * 16 * DT;
        static_assert((WK - 1) * WM * PIECE * 4 <= 4 * TILE_B, "the join uses the tiles' memory");
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
    if (a.pq) {
        const long rid = ((long)at.b * rw.M + at.i) * ((long)rw.Hk * rw.G) + at.h;
        float *p = a.pq + ((long)split * ((long)rw.grid_b * rw.M * rw.Hk * rw.G) + rid) * rw.D;
        store_column<float, DT>(p, dq, rw.D, half, at.exists, [=](float x) { return weights ? x : 0.0f; });
        return;
    }
    store_column<T, DT>((T *)a.dq + at.b * a.dqb + at.i * a.dqr + at.h * a.dqh, dq, rw.D, half, at.exists,
                        [&](float x) { return weights ? x * a.scale : 0.0f; });
}

// dK, dV: two waves per SIMD at 128 features of 16 bits (241 registers, fp16 245; one wave with 372 registers took 1767 us where this
// takes 1010 to 1061).  4 waves of 32 keys each; the rows pass through LDS in tiles of BR.  S = Q K^T and dP = dO V^T with a lane holding
// one key, then dV^T += dO^T P and dK^T += Q^T dS.
// OWN: in one launch with dQ; <dO, O> is formed here, from tiles of O beside those of dO, once per tile by all threads.
template <typename T, int DT, bool OWN>
__device__ __forceinline__ void attend_dkv_block(const AttendBwd &a, char *lds, float *stat, unsigned id, unsigned total)
{
    using TL = Tile<T, DT>;
    constexpr int BR = attend_dkv_br(sizeof(T));
    using FL = Fill<T, DT, BR>;
    constexpr int TILE_B = BR * TL::ROWB, STAGE_B = (OWN ? 3 : 2) * TILE_B;
    // lds: [stage][Q, dO (, O)]; stat: [stage][lse, <dO, O>][64] (OWN: lse as it is in memory), OWN: then lse in log2 units and <dO, O>
    float *own = stat + 4 * 64;

    // 128 features fill the registers: what follows from the lane's number is formed again where it is needed, not kept
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto lane_again = [] {
        int x = threadIdx.x & 63;
        asm volatile("" : "+v"(x));
        return x;
    };
    const AttendRows &rw = a.rows;
    int ktile, u;
    place_block(id, total, a.k_order, a.ktiles, a.by_ktiles, ktile, u);
    const int us = rw.by_hk(u), hk = u - us * rw.Hk;
    const int turn = a.by_k_splits(us), split = us - turn * a.k_splits;
    const int bz = nth_longest(a.keys, rw.grid_b, turn);

    const int len = clamped(a.keys.len, bz, a.keys.n);
    const auto counts_of = [&](int key) { return key < len && (!a.keys.mask || a.keys.mask[bz * a.keys.mask_b + key]); };
    const int key0 = ktile * ATTEND_DKV_KEYS + wave * 32;
    // rows are packed (query, head of the group); queries from q_len on do not count
    const int begin = split * a.k_chunk;
    const int end = ktile * ATTEND_DKV_KEYS < len ? min(clamped(rw.len, bz, rw.M) * rw.G, begin + a.k_chunk) : 0;

    const unsigned lds0 = lds_offset(lds), stat0 = lds_offset(stat);
    const int h0 = hk * rw.G;
    const T *qp = (const T *)rw.q + bz * rw.qb + h0 * rw.qh, *gp = (const T *)a.dout + bz * a.gb + h0 * a.gh;
    const T *op = (const T *)a.o + bz * a.ob + h0 * a.oh;
    const float *sp = (OWN ? a.lse : a.stat) + ((long)bz * rw.Hk * rw.G + h0) * rw.M;
    const long stats = (long)rw.grid_b * rw.Hk * rw.G * rw.M;
    const unsigned qrb = (unsigned)(rw.qr * sizeof(T)), qhb = (unsigned)(rw.qh * sizeof(T));
    const unsigned grb = (unsigned)(a.gr * sizeof(T)), ghb = (unsigned)(a.gh * sizeof(T));
    const unsigned orb = (unsigned)(a.orow * sizeof(T)), ohb = (unsigned)(a.oh * sizeof(T));
    const auto fetch = [&](int r0, int stage) {
        const int n0 = rw.by_g(r0), lane = lane_again();
        const u32x4 qd = dma_buffer(qp + (long)n0 * rw.qr, DMA_MOST), gd = dma_buffer(gp + (long)n0 * a.gr, DMA_MOST);
        u32x4 od;
        if constexpr (OWN)
            od = dma_buffer(op + (long)n0 * a.orow, DMA_MOST);
        const unsigned at0 = lds0 + stage * STAGE_B;
#pragma unroll(DT > 2 ? 1 : FL::N)
        for (int x = 0; x < FL::N; ++x)
            if (FL::on(x, wave)) {
                const int r = r0 + FL::row(x, wave, lane);
                const int n = rw.by_g(r), g = r - n * rw.G;
                const unsigned c = FL::chunk(x, wave, lane, rw.D);
                const bool off = r >= end || c == DMA_OUT;
                dma16(qd, off ? DMA_OUT : (unsigned)(n - n0) * qrb + g * qhb + c, at0 + FL::lds(x, wave));
                dma16(gd, off ? DMA_OUT : (unsigned)(n - n0) * grb + g * ghb + c, at0 + TILE_B + FL::lds(x, wave));
                if constexpr (OWN)
                    dma16(od, off ? DMA_OUT : (unsigned)(n - n0) * orb + g * ohb + c, at0 + 2 * TILE_B + FL::lds(x, wave));
            }
        if (wave < (OWN ? 1 : 2)) {  // a row past the end gets zeros, and has zeros for Q and dO: it adds nothing
            const int r = r0 + lane;
            const int n = rw.by_g(r), g = r - n * rw.G;
            const u32x4 sd = dma_buffer(sp + wave * stats + n0, DMA_MOST);
            dma4(sd, lane < BR && r < end ? 4u * (g * rw.M + (n - n0)) : DMA_OUT, stat0 + (stage * 2 + wave) * 256);
        }
    };
    if (begin < end)
        fetch(begin, 0);

    Frag<T> kf[2 * DT], vf[2 * DT];
    {
        const int lane = lane_again(), key = key0 + (lane & 31);
        const bool counts = counts_of(key);
        load_row_frags<T, DT>(kf, (const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh + (counts ? key * a.keys.kr : 0), counts, rw.D, lane);
        load_row_frags<T, DT>(vf, (const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh + (counts ? key * a.keys.vr : 0), counts, rw.D, lane);
    }

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            dk[d][i] = dv[d][i] = 0.0f;
    float f = F_START;  // (NARROW)

    int stage = 0;
    for (int r0 = begin; r0 < end; r0 += BR, stage ^= 1) {
        dma_wait();
        __syncthreads();
        if (r0 + BR < end)
            fetch(r0 + BR, stage ^ 1);
        if constexpr (OWN) {  // P threads of consecutive lanes to a row, every P-th chunk each
            constexpr int P = 256 / BR;
            const int tid = wave * 64 + lane_again(), row = tid / P, part = tid % P;
            const char *gt = lds + stage * STAGE_B + TILE_B, *ot = gt + TILE_B;
            float s = 0.0f;
#pragma unroll
            for (int c = part; c < TL::LC; c += P) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(gt + row * TL::ROWB + 16 * c), y = *reinterpret_cast<const u32x4 *>(ot + row * TL::ROWB + 16 * c);
                typedef T vec __attribute__((ext_vector_type(TL::EPC)));
                const vec g = __builtin_bit_cast(vec, x), o = __builtin_bit_cast(vec, y);
#pragma unroll
                for (int j = 0; j < TL::EPC; ++j)
                    s += (float)g[j] * (float)o[j];
            }
#pragma unroll
            for (int k = P / 2; k; k >>= 1)
                s += __shfl_xor(s, k);
            if (part == 0) {
                const float lse = stat[stage * 2 * 64 + row];
                const bool none = lse == NEG_INF;  // (a row past the end: 0, with zeros for Q and dO)
                own[row] = none ? POS_INF : lse * 1.44269504088896f - P_LIFT<T>;
                own[64 + row] = none ? 0.0f : s;
            }
            __syncthreads();
        }
        const float *sl = OWN ? own : stat + stage * 2 * 64, *sd = sl + 64;
#pragma unroll 1
        for (int s = 0; s < BR / 32; ++s) {
            const int lane = lane_again(), half = lane >> 5, at0 = stage * STAGE_B + s * 32 * TL::ROWB;
            const int rbase = TL::row_base(lane) + at0, cbase = TL::col_base(lane) + at0;
            const char *qt = lds, *gt = lds + TILE_B;
            f32x16 p, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                p[i] = dp[i] = 0.0f;
#pragma unroll
            for (int t = 0; t < TL::KS; ++t) {
                p = mma(TL::row_frag(qt, rbase, 0, t), kf[t], p);
                dp = mma(TL::row_frag(gt, rbase, 0, t), vf[t], dp);
            }
            __builtin_amdgcn_sched_barrier(0);  // the statistics' registers only from here on
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 ls = *reinterpret_cast<const f32x4 *>(sl + 32 * s + 8 * x + 4 * half);
                const f32x4 ds = *reinterpret_cast<const f32x4 *>(sd + 32 * s + 8 * x + 4 * half);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 4 * x + j;
                    p[i] = exp2_(p[i] * a.c - ls[j]);
                    dp[i] = p[i] * (dp[i] - ds[j]);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Frag<T> w = as_operand<T>(p, t);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    dv[d] = mma(TL::col_frag(gt, cbase, 16 * t, d), w, dv[d]);
            }
            if constexpr (NARROW<T>) {
                const float top = largest(dp) * f;
                if (__any(top > F_MOST)) {
                    const float g = bring_down(top);
                    f *= g;
                    times<DT>(dk, g);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    dp[i] *= f;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Frag<T> w = as_operand<T>(dp, t);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    dk[d] = mma(TL::col_frag(qt, cbase, 16 * t, d), w, dk[d]);
            }
        }
    }
    const int lane = lane_again(), half = lane >> 5, key = key0 + (lane & 31);
    const bool exists = key < a.keys.n, counts = exists && counts_of(key);
    if constexpr (NARROW<T>) {
        times<DT>(dk, reciprocal_of_power(f) * 0x1p-12f);
        times<DT>(dv, 0x1p-12f);
    }
    // a key that does not count had zeros for its features: its sums are of finite weights but not zero
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            dk[d][i] = counts ? dk[d][i] : 0.0f;
            dv[d][i] = counts ? dv[d][i] : 0.0f;
        }
    const auto same = [](float x) { return x; };
    if (a.pk) {
        const long at = ((long)split * rw.grid_b * rw.Hk + (long)bz * rw.Hk + hk) * a.keys.n + key;
        store_column<float, DT>(a.pk + at * rw.D, dk, rw.D, half, exists, same);
        store_column<float, DT>(a.pv + at * rw.D, dv, rw.D, half, exists, same);
        return;
    }
    store_column<T, DT>((T *)a.dk + bz * a.dkb + key * a.dkr + hk * a.dkh, dk, rw.D, half, exists, [&](float x) { return x * a.scale; });
    store_column<T, DT>((T *)a.dv + bz * a.dvb + key * a.dvr + hk * a.dvh, dv, rw.D, half, exists, same);
}

// the kernel's argument (its only one) where it lies
__device__ __forceinline__ const AttendBwd &args_again()
{
    typedef const __attribute__((address_space(4))) AttendBwd *arg;
    arg p = (arg)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttendBwd *)p;
}
template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (attend_dq_per_cu(sizeof(T), DT, WM))) void attend_dq_kernel(AttendBwd a)
{
    __shared__ __attribute__((aligned(1024))) char lds[attend_dq_lds(sizeof(T), DT, WM)];
    __shared__ __attribute__((aligned(16))) float bias[2 * attend_dq_bn(WM)];
    attend_dq_block<T, DT, WM>(a, lds, bias, blockIdx.x, gridDim.x);
}
template <typename T, int DT>
__global__ __launch_bounds__(256, (attend_dkv_per_cu(sizeof(T), DT))) void attend_dkv_kernel(AttendBwd a)
{
    __shared__ __attribute__((aligned(1024))) char lds[attend_dkv_lds(sizeof(T), DT, false)];
    __shared__ __attribute__((aligned(1024))) float stat[4 * 64];
    attend_dkv_block<T, DT, false>(a, lds, stat, blockIdx.x, gridDim.x);
}
// Both in one launch: where neither fills the card by itself.
template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (attend_both_per_cu(sizeof(T), DT, WM))) void attend_both_kernel(AttendBwd a)
{
    constexpr int A = attend_dq_lds(sizeof(T), DT, WM), B = attend_dkv_lds(sizeof(T), DT, true);
    __shared__ __attribute__((aligned(1024))) char lds[A > B ? A : B];
    __shared__ __attribute__((aligned(1024))) float small[6 * 64];
    static_assert(2 * attend_dq_bn(WM) <= 6 * 64, "bias and statistics share their place");
    // Each side reads the arguments for itself: what both need, loaded once in front of the branch, would not fit the scalar registers.
    const unsigned n = a.ktiles * a.k_splits * a.rows.Hk * a.rows.grid_b;
    if (blockIdx.x < n)
        attend_dkv_block<T, DT, true>(args_again(), lds, small, blockIdx.x, n);
    else
        attend_dq_block<T, DT, WM>(args_again(), lds, small, blockIdx.x - n, gridDim.x - n);
}

// out[row] = f sum_s p[s][row], in slot order; rows of D values, four per lane.  Row -> (batch, n, head) by the strides.  Up to
// three of them (dQ, dK, dV) in one launch.
struct AttendSum {
    const float *p = nullptr;
    int slots = 0, n = 1, H = 1;  // row = (b n + i) H + h or, head_first, (b H + h) n + i
    long rows = 0;
    int head_first = 0;
    float f = 1;
    void *out = nullptr;
    long ob = 0, orow = 0, oh = 0;
    unsigned blocks = 0;
};
struct AttendSums {
    AttendSum s[3];
    int D;
};
template <typename T>
__global__ __launch_bounds__(256) void attend_sum_kernel(AttendSums all)
{
    unsigned at = blockIdx.x;
    int w = 0;
    while (w < 2 && at >= all.s[w].blocks)
        at -= all.s[w++].blocks;
    const AttendSum &a = all.s[w];
    const int q = all.D >> 2;
    const long id = (long)at * 256 + threadIdx.x;
    if (id >= a.rows * q)
        return;
    const long row = id / q;
    const int d = 4 * (int)(id - row * q);
    f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
    for (int k = 0; k < a.slots; ++k)
        s += *reinterpret_cast<const f32x4 *>(a.p + ((long)k * a.rows + row) * all.D + d);
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
    x4<T> v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = (T)(s[j] * a.f);
    *reinterpret_cast<x4<T> *>((T *)a.out + b * a.ob + i * a.orow + h * a.oh + d) = v;
}

template <typename T, int DT, int WM>
void launch_bwd_shape(const AttendBwd &a, hipStream_t st)
{
    const unsigned nq = (unsigned)(a.mtiles * a.q_splits * a.rows.Hk * a.rows.grid_b), nk = (unsigned)(a.ktiles * a.k_splits * a.rows.Hk * a.rows.grid_b);
    if (a.fused) {
        hipLaunchKernelGGL((attend_both_kernel<T, DT, WM>), dim3(nq + nk), dim3(256), 0, st, a);
        return;
    }
    if (a.rows.R > 0)
        hipLaunchKernelGGL((attend_dq_kernel<T, DT, WM>), dim3(nq), dim3(256), 0, st, a);
    if (a.keys.n > 0)
        hipLaunchKernelGGL((attend_dkv_kernel<T, DT>), dim3(nk), dim3(256), 0, st, a);
}
template <typename T, int DT>
void launch_bwd_dim(const AttendBwd &a, hipStream_t st)
{
    switch (a.wm) {
    case 1:
        if constexpr (attend_least_wm(sizeof(T), DT) == 1)
            launch_bwd_shape<T, DT, 1>(a, st);
        break;
    case 2: launch_bwd_shape<T, DT, 2>(a, st); break;
    default: launch_bwd_shape<T, DT, 4>(a, st); break;
    }
}

}  // namespace attend

template <typename T>
void attend_launch_bwd(const AttendBwd &a, hipStream_t st)
{
    const AttendRows &rw = a.rows;
    switch (attend_dt(rw.D)) {
    case 1: attend::launch_bwd_dim<T, 1>(a, st); break;
    case 2: attend::launch_bwd_dim<T, 2>(a, st); break;
    case 3: attend::launch_bwd_dim<T, 3>(a, st); break;
    default: attend::launch_bwd_dim<T, 4>(a, st); break;
    }
    attend::AttendSums s;
    s.D = rw.D;
    if (a.pq) {
        attend::AttendSum &q = s.s[0];
        q.p = a.pq, q.slots = a.q_splits, q.n = rw.M, q.H = rw.Hk * rw.G, q.rows = (long)rw.grid_b * rw.M * q.H, q.f = a.scale;
        q.out = a.dq, q.ob = a.dqb, q.orow = a.dqr, q.oh = a.dqh;
    }
    if (a.pk) {
        attend::AttendSum &k = s.s[1], &v = s.s[2];
        k.slots = a.k_splits, k.n = a.keys.n, k.H = rw.Hk, k.rows = (long)rw.grid_b * rw.Hk * a.keys.n, k.head_first = 1;
        v = k;
        k.p = a.pk, k.f = a.scale, k.out = a.dk, k.ob = a.dkb, k.orow = a.dkr, k.oh = a.dkh;
        v.p = a.pv, v.out = a.dv, v.ob = a.dvb, v.orow = a.dvr, v.oh = a.dvh;
    }
    unsigned grid = 0;
    for (attend::AttendSum &x : s.s)
        grid += x.blocks = (unsigned)((x.rows * (rw.D / 4) + 255) / 256);
    if (grid)
        hipLaunchKernelGGL((attend::attend_sum_kernel<T>), dim3(grid), dim3(256), 0, st, s);
}

}  // namespace gpx
