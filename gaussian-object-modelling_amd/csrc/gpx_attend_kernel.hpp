// gpx_attend_kernel.hpp -- the kernels of gpx_attend / gpx_attend_shared (forward) and gpx_attend_backward, as templates over
// the element type; gpx_attend_f32.hip, _f16.hip and _bf16.hip instantiate them.
#pragma once
#include "gpx_attend_tile.hpp"

namespace gpx {
namespace attend {

// ---- forward -----------------------------------------------------------------------------------------------------------------
// One workgroup of 4 waves: WM waves along the rows (32 packed rows each), WK = 4 / WM along the keys.  Scores are formed
// TRANSPOSED, S^T = K Q^T: a lane then holds one row's weights (its column), the running maximum and sum of a row are one
// register per lane, and S^T turns into the operand of O^T = V^T P^T without leaving the lane (gpx_attend_tile.hpp).
// Keys and values are read from memory once per 32 WM rows, as tiles of BN rows, two of them in LDS: while one is worked on the
// next is on its way.
template <typename T, int DT, int WM>
struct FwdShape {
    static constexpr int WK = 4 / WM;
    static constexpr int KT = sizeof(T) == 2 && WK == 1 ? 64 : 32;  // keys of a wave per step
    static constexpr int BN = KT * WK;
    static constexpr int BM = 32 * WM;
    static constexpr int LDS = 4 * BN * Tile<T, DT>::ROWB;
    // workgroups a CU has room for (its 160 KB of LDS, and two waves per SIMD where the registers allow it)
    static constexpr int PER_CU = LDS <= 80 * 1024 - 1024 ? 2 : 1;
};

template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (FwdShape<T, DT, WM>::PER_CU)) void attend_fwd_kernel(AttendFwd a)
{
    using TL = Tile<T, DT>;
    using SH = FwdShape<T, DT, WM>;
    constexpr int BN = SH::BN, WK = SH::WK, KT = SH::KT, NS = KT / 32;
    using FL = Fill<T, DT, BN>;
    constexpr int TILE_B = BN * TL::ROWB;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B];  // [stage][keys, values]
    __shared__ __attribute__((aligned(16))) float bias[2][BN];       // 0, or -inf where the key does not count

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;
    const AttendRows &rw = a.rows;
    const int mtiles = (rw.R + SH::BM - 1) / SH::BM;
    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    const int mt = id % mtiles;
    id /= mtiles;
    const int split = id % a.splits;
    id /= a.splits;
    const int hk = id % rw.Hk, bz = id / rw.Hk;

    const RowAt at = row_at(rw, bz, hk, mt * SH::BM + wm * 32 + (lane & 31));
    const int len = clamped(a.keys.len, bz, a.keys.n);
    const int begin = split * a.chunk, end = min(len, begin + a.chunk);
    const int upto = a.tail ? len - (rw.M - 1 - at.i) : len;  // keys this row may see

    const unsigned ksb = (unsigned)(a.keys.kr * sizeof(T)), vsb = (unsigned)(a.keys.vr * sizeof(T));  // row strides, bytes
    const char *kp = (const char *)((const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh);
    const char *vp = (const char *)((const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh);
    const unsigned char *mask = a.keys.mask ? a.keys.mask + bz * a.keys.mask_b : nullptr;
    const unsigned lds0 = lds_offset(lds);

    unsigned ko[FL::N], vo[FL::N];  // the lane's places in a tile, as offsets from its first row
#pragma unroll
    for (int x = 0; x < FL::N; ++x) {
        const unsigned c = FL::chunk(x, wave, lane, rw.D), r = FL::row(x, wave, lane);
        ko[x] = c == DMA_OUT ? DMA_OUT : r * ksb + c;
        vo[x] = c == DMA_OUT ? DMA_OUT : r * vsb + c;
    }
    // mask bytes of the tile after the next: for the rows the lane fetches, and (bit 8) for the key it writes the bias of
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
#pragma unroll
        for (int x = 0; x < FL::N; ++x)
            if (FL::on(x, wave)) {
                const bool off = mask && !mb[x];
                dma16(kd, off ? DMA_OUT : ko[x], at0 + FL::lds(x, wave));
                dma16(vd, off ? DMA_OUT : vo[x], at0 + TILE_B + FL::lds(x, wave));
            }
        if (tid < BN && (mask || n0 + BN > end))
            bias[stage][tid] = n0 + tid < end && (!mask || mb[FL::N]) ? 0.0f : NEG_INF;
    };
    if (begin < end) {
        look(begin);
        fetch(begin, 0);
        look(begin + BN);
    }

    x8<T> qf[2 * DT];
    load_row_frags<T, DT>(qf, (const T *)rw.q + (at.valid ? at.b * rw.qb + at.i * rw.qr + at.h * rw.qh : 0), at.valid, rw.D, lane);

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            o[d][i] = 0.0f;
    float m = NEG_INF, l = 0.0f;

    int stage = 0;
    for (int n0 = begin; n0 < end; n0 += BN, stage ^= 1) {
        dma_wait();
        __syncthreads();  // this tile is there, and nobody reads the other one any more
        if (n0 + BN < end) {
            fetch(n0 + BN, stage ^ 1);
            look(n0 + 2 * BN);
        }
        const char *kt = lds + stage * 2 * TILE_B, *vt = kt + TILE_B;
        const int rbase = TL::row_base(lane), cbase = TL::col_base(lane);
        const int w0 = n0 + wk * KT;

        // a key that does not count starts at -inf (its features are zeros) and stays there
        f32x16 sc[NS];
        if (mask || n0 + BN > end) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 w = *reinterpret_cast<const f32x4 *>(&bias[stage][wk * KT + 32 * s + 8 * x + 4 * half]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[s][4 * x + j] = w[j];
                }
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[s][i] = 0.0f;
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < TL::KS; ++t)
                sc[s] = mma(TL::row_frag(kt, rbase, wk * KT + 32 * s, t), qf[t], sc[s]);
        if (a.tail && w0 + KT > len - rw.M + 1) {  // keys that only some of the rows see
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int left = upto - (w0 + 32 * s);
                const unsigned bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[s][i] = bit_of(bits, half, i) ? sc[s][i] : NEG_INF;
            }
        }
        float top = NEG_INF;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                top = fmaxf(top, sc[s][i]);
        top = fmaxf(top, other_half(top)) * a.c;
        // The running maximum need not be the true one: sums in 32 bits and weights of up to 2^8 lose nothing, so it is
        // raised (and what is summed so far rescaled) only when the new one is more than 8 above it.
        if (__any(top > m + 8.0f || (m == NEG_INF && top > NEG_INF))) {
            const float mn = fmaxf(m, top);
            const float f = mn == NEG_INF ? 1.0f : exp2_(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[d][i] *= f;
        }
        const float sub = m == NEG_INF ? 0.0f : m;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[s][i] = exp2_(sc[s][i] * a.c - sub);
                l += sc[s][i];
            }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const x8<T> p = as_operand<T>(sc[s], t);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = mma(TL::col_frag(vt, cbase, wk * KT + 32 * s + 16 * t, d), p, o[d]);
            }
    }
    l += other_half(l);

    if constexpr (WK > 1) {  // join the waves' pieces of the key range, in wave order
        constexpr int PIECE = 64 * 16 * DT + 128;
        static_assert((WK - 1) * WM * PIECE * 4 <= 4 * TILE_B, "the join uses the tiles' memory");
        float *pc = reinterpret_cast<float *>(lds);
        __syncthreads();
        if (wk > 0) {
            float *w = pc + ((wk - 1) * WM + wm) * PIECE;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    w[(d * 16 + i) * 64 + lane] = o[d][i];
            w[64 * 16 * DT + lane] = m;
            w[64 * 16 * DT + 64 + lane] = l;
        }
        __syncthreads();
        if (wk > 0)
            return;
#pragma unroll
        for (int k = 1; k < WK; ++k) {
            const float *w = pc + ((k - 1) * WM + wm) * PIECE;
            const float mo = w[64 * 16 * DT + lane], lo = w[64 * 16 * DT + 64 + lane];
            const float mn = fmaxf(m, mo);
            const float f0 = m == NEG_INF ? 0.0f : exp2_(m - mn), f1 = mo == NEG_INF ? 0.0f : exp2_(mo - mn);
            l = l * f0 + lo * f1;
            m = mn;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[d][i] = o[d][i] * f0 + w[(d * 16 + i) * 64 + lane] * f1;
        }
    }
    if (!at.exists)
        return;
    const long rid = ((long)at.b * rw.M + at.i) * ((long)rw.Hk * rw.G) + at.h;
    if (!at.valid)
        m = NEG_INF, l = 0.0f;
    if (a.po) {
        const long slot = (long)(a.slot0 + split) * a.slot_rows + rid;
        if (half == 0)
            a.pml[slot] = make_float2(m, l);
        if (l == 0.0f)
            return;  // a piece without weights is never read
        float *po = a.po + slot * rw.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int f = 32 * d + 8 * x + 4 * half;
                if (f < rw.D)
                    *reinterpret_cast<f32x4 *>(po + f) = f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
            }
        return;
    }
    if (half == 0)
        a.lse[((long)at.b * rw.Hk * rw.G + at.h) * rw.M + at.i] = l == 0.0f ? NEG_INF : (m + log2_(l)) * 0.693147180559945f;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const bool none = l == 0.0f;
    T *po = (T *)a.o + at.b * a.ob + at.i * a.orow + at.h * a.oh;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int f = 32 * d + 8 * x + 4 * half;
            x4<T> w;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = none ? (T)0.0f : (T)(o[d][4 * x + j] * inv);
            if (f < rw.D)
                *reinterpret_cast<x4<T> *>(po + f) = w;
        }
}

// One wave per row: the pieces' maxima and sums (a lane each, 64 at a time), then the pieces' sums weighted by them.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendJoin a)
{
    const int lane = threadIdx.x & 63;
    const long rid = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rid >= a.slot_rows)
        return;
    float top = NEG_INF;
    for (int s = lane; s < a.slots; s += 64)
        top = fmaxf(top, a.pml[s * a.slot_rows + rid].x);
#pragma unroll
    for (int k = 32; k; k >>= 1)
        top = fmaxf(top, __shfl_xor(top, k));
    const int d = 2 * lane;  // D is at most 128
    float l = 0.0f, x = 0.0f, y = 0.0f;
    for (int s0 = 0; s0 < a.slots; s0 += 64) {
        float w = 0.0f;
        if (s0 + lane < a.slots) {
            const float2 ml = a.pml[(long)(s0 + lane) * a.slot_rows + rid];
            w = ml.y == 0.0f ? 0.0f : exp2_(ml.x - top);
            l += ml.y == 0.0f ? 0.0f : w * ml.y;
        }
        const int k = min(64, a.slots - s0);
        for (int s = 0; s < k; ++s) {
            const float ws = __shfl(w, s);
            if (ws != 0.0f && d < a.D) {
                const float2 p = *reinterpret_cast<const float2 *>(a.po + ((s0 + s) * a.slot_rows + rid) * a.D + d);
                x += ws * p.x;
                y += ws * p.y;
            }
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1)
        l += __shfl_xor(l, k);
    const int h = (int)(rid % a.H);
    const long n = rid / a.H;
    const int i = (int)(n % a.M);
    const long b = n / a.M;
    const bool none = l == 0.0f;
    if (lane == 0)
        a.lse[(b * a.H + h) * a.M + i] = none ? NEG_INF : (top + log2_(l)) * 0.693147180559945f;
    if (d < a.D) {
        T *o = (T *)a.o + b * a.ob + i * a.orow + h * a.oh + d;
        const float inv = none ? 0.0f : 1.0f / l;
        o[0] = none ? (T)0.0f : (T)(x * inv);
        o[1] = none ? (T)0.0f : (T)(y * inv);
    }
}

template <typename T, int DT, int WM>
void launch_fwd_shape(const AttendFwd &a, hipStream_t st)
{
    const int mtiles = (a.rows.R + 32 * WM - 1) / (32 * WM);
    const unsigned grid = (unsigned)((long)mtiles * a.splits * a.rows.Hk * a.rows.grid_b);
    hipLaunchKernelGGL((attend_fwd_kernel<T, DT, WM>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T, int DT>
void launch_fwd_dim(const AttendFwd &a, hipStream_t st)
{
    switch (attend_block_rows(sizeof(T) == 4, a.rows.D, a.rows.R)) {
    case 32:
        if constexpr (sizeof(T) == 2 || DT <= 2)
            launch_fwd_shape<T, DT, 1>(a, st);
        break;
    case 64: launch_fwd_shape<T, DT, 2>(a, st); break;
    default: launch_fwd_shape<T, DT, 4>(a, st); break;
    }
}

}  // namespace attend

template <typename T>
void attend_launch_fwd(const AttendFwd &a, hipStream_t st)
{
    switch ((a.rows.D + 31) / 32) {
    case 1: return attend::launch_fwd_dim<T, 1>(a, st);
    case 2: return attend::launch_fwd_dim<T, 2>(a, st);
    case 3: return attend::launch_fwd_dim<T, 3>(a, st);
    default: return attend::launch_fwd_dim<T, 4>(a, st);
    }
}
template <typename T>
void attend_launch_join(const AttendJoin &a, hipStream_t st)
{
    hipLaunchKernelGGL((attend::attend_join_kernel<T>), dim3((unsigned)((a.slot_rows + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace gpx
