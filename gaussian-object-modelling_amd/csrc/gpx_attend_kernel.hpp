// gpx_attend_kernel.hpp -- the kernels of gpx_attend / gpx_attend_shared (forward) and gpx_attend_backward, as templates over
// the element type; gpx_attend_f32.hip, _f16.hip and _bf16.hip instantiate them.
#pragma once
#include <type_traits>

#include "gpx_attend_tile.hpp"

namespace gpx {
namespace attend {

// ---- forward -----------------------------------------------------------------------------------------------------------------
// o_i = sum_j 2^(c s_ij - m_i) v_j / sum_j 2^(c s_ij - m_i), s = Q K^T, c = scale log2(e), in one pass over the keys with a running
// maximum m and sum l per row.
// One workgroup of 4 waves: WM waves along the rows (32 packed rows each), WK = 4 / WM along the keys.  Scores are formed
// TRANSPOSED, S^T = K Q^T: a lane then holds one row's weights (its column), the running maximum and sum of a row are one
// register per lane, and S^T turns into the operand of O^T = V^T P^T without leaving the lane (gpx_attend_tile.hpp).
// Keys and values are read from memory once per 32 WM rows, as tiles of BN rows, two of them in LDS: while one is worked on the
// next is on its way.  64 keys a wave and step for the 16-bit types with WM = 4 (32: as fast at 64 and slower at 96 features).
// What bounds it (bf16; the library's 8192^3 product reaches 1067 TFLOP/s on the same card):
//   16384 x 16384, 16 heads of 128   2.06 to 2.15 ms from card to card, 1066 to 1023 TFLOP/s: the matrix cores at the card's power limit
//                                    (clock 1.9-2.1 GHz; without the softmax 2.01, without any fetch 1.95)
//   32768 x 724, 8 heads of 64       67 us, 724 TFLOP/s: neither vector issue (59 % of the SIMDs' time; 156 instructions a tile and wave,
//                                    128 of them the softmax's) nor matrix cores (31 %) are full: 2048 workgroups of 12 tiles on
//                                    768 places are 2.7 rounds paid as three, each with its own start and end
//   4 x 65536, 32/8 heads of 128 x 3 156 us, 5.2 TB/s: memory
// STAGES == 1 has one tile at a time (the own part of a shared call: short ranges, many workgroups a CU).
// fp16 has normal numbers from 2^-14 to 2^15 only: its weights are rounded as 2^LIFT of what they are relative to m, so that an entry
// 2^-21 of the row's largest still has all its bits (and one of 2^-31 some): many of them can be most of a long context's sum.  The
// factor is in m, so sums, joins and lse need no other form, and with the lag of 8 below weights stay at or under 2^15.
template <typename T> constexpr float WEIGHT_LIFT = std::is_same_v<T, _Float16> ? 7.0f : 0.0f;
template <typename T, int DT, int WM, int STAGES>
__device__ __forceinline__ void attend_fwd_block(const AttendFwd &a, char *lds, float *bias, unsigned id, unsigned total)
{
    using TL = Tile<T, DT>;
    constexpr int WK = 4 / WM, KT = attend_fwd_kt(sizeof(T), DT, WM), NS = KT / 32, BN = KT * WK;
    using FL = Fill<T, DT, BN>;
    constexpr float LIFT = WEIGHT_LIFT<T>;
    constexpr int TILE_B = BN * TL::ROWB;  // lds: [stage][keys, values]; bias: [stage][BN], 0 or -inf where the key does not count

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wm = wave % WM, wk = wave / WM;
    const AttendRows &rw = a.rows;
    int mt, u;
    place_block(id, total, a.order, a.mtiles, a.by_mtiles, mt, u);
    const int us = rw.by_hk(u), hk = u - us * rw.Hk;
    const int turn = a.by_splits(us), split = us - turn * a.splits;
    const int bz = nth_longest(a.keys, rw.grid_b, turn);

    const RowAt at = row_at(rw, bz, hk, mt * 32 * WM + wm * 32 + (lane & 31));
    const int len = clamped(a.keys.len, bz, a.keys.n);
    const int begin = split * a.chunk, end = min(len, begin + a.chunk);
    const int upto = a.tail ? len - (rw.M - 1 - at.i) : len;  // keys this row may see

    const unsigned ksb = (unsigned)(a.keys.kr * sizeof(T)), vsb = (unsigned)(a.keys.vr * sizeof(T));  // row strides, bytes
    const char *kp = (const char *)((const T *)a.keys.k + bz * a.keys.kb + hk * a.keys.kh);
    const char *vp = (const char *)((const T *)a.keys.v + bz * a.keys.vb + hk * a.keys.vh);
    const unsigned char *mask = a.keys.mask ? a.keys.mask + bz * a.keys.mask_b : nullptr;
    const unsigned lds0 = lds_offset(lds);

    // the lane's places in a tile, as offsets from its first row: kept, or formed at every tile where registers are short
    constexpr bool KEEP = sizeof(T) == 2 || DT <= 2;
    unsigned ko[KEEP ? FL::N : 1], vo[KEEP ? FL::N : 1];
    const auto place = [&](int x, int ln, unsigned &k, unsigned &v) {
        const unsigned c = FL::chunk(x, wave, ln, rw.D), r = FL::row(x, wave, ln);
        k = c == DMA_OUT ? DMA_OUT : r * ksb + c;
        v = c == DMA_OUT ? DMA_OUT : r * vsb + c;
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int x = 0; x < FL::N; ++x)
            place(x, lane, ko[x], vo[x]);
    }
    // mask bytes of the next tile to fetch: for the rows the lane fetches, and for the key it writes the bias of
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
        int ln = lane;
        if constexpr (!KEEP)
            asm volatile("" : "+v"(ln));
#pragma unroll
        for (int x = 0; x < FL::N; ++x)
            if (FL::on(x, wave)) {
                unsigned k, v;
                if constexpr (KEEP)
                    k = ko[x], v = vo[x];
                else
                    place(x, ln, k, v);
                if (mask) {
                    k = mb[x] ? k : DMA_OUT;
                    v = mb[x] ? v : DMA_OUT;
                }
                dma16(kd, k, at0 + FL::lds(x, wave));
                dma16(vd, v, at0 + TILE_B + FL::lds(x, wave));
            }
        if ((mask || a.tail || n0 + BN > end) && tid < BN)
            bias[stage * BN + tid] = n0 + tid < end && (!mask || mb[FL::N]) ? 0.0f : NEG_INF;
    };
    if (begin < end) {
        look(begin);
        fetch(begin, 0);
        look(begin + BN);
    }

    Frag<T> qf[2 * DT];
    load_row_frags<T, DT>(qf, (const T *)rw.q + (at.valid ? at.b * rw.qb + at.i * rw.qr + at.h * rw.qh : 0), at.valid, rw.D, lane);

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            o[d][i] = 0.0f;
    float m = NEG_INF, l = 0.0f;

    // one tile; EDGE: some of its keys do not count, or not for every row
    const auto step = [&](int n0, int stage, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        const char *kt = lds, *vt = lds + TILE_B;
        const int rbase = TL::row_base(lane) + stage * 2 * TILE_B, cbase = TL::col_base(lane) + stage * 2 * TILE_B;
        f32x16 sc[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[s][i] = 0.0f;
            if constexpr (EDGE) {  // a key that does not count starts at -inf (its features are zeros) and stays there
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 w = *reinterpret_cast<const f32x4 *>(&bias[stage * BN + wk * KT + 32 * s + 8 * x + 4 * half]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[s][4 * x + j] = w[j];
                }
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < TL::KS; ++t)
                sc[s] = mma(TL::row_frag(kt, rbase, wk * KT + 32 * s, t), qf[t], sc[s]);
        if constexpr (EDGE) {
            const int w0 = n0 + wk * KT;
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
        }
        float top = NEG_INF;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                top = fmaxf(top, sc[s][i]);
        top = max_both_halves(top) * a.c;
        // The running maximum m + LIFT need not be the true one: sums in 32 bits and weights of up to 2^8 (times 2^LIFT) lose
        // nothing, so it is raised (and what is summed so far rescaled) only when the new one is more than 8 above it.  (A row
        // without a key so far has m = -inf, and is raised by any.)
        if (__any(top > m + (8.0f + LIFT))) {
            const float mn = fmaxf(m, top - LIFT);
            const float f = mn == NEG_INF ? 1.0f : exp2_(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[d][i] *= f;
        }
        const float sub = m == NEG_INF ? 0.0f : m;  // (no key that counts so far, or only scores below the fp32 range: weights 0)
        // The tile's weights are added up before they join l: one at a time, weights 2^-25 of l and less would leave it as it is,
        // however many there are.
        float add = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[s][i] = exp2_(sc[s][i] * a.c - sub);
                add = s == 0 && i == 0 ? sc[s][i] : add + sc[s][i];
            }
        l += add;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Frag<T> p = as_operand<T>(sc[s], t);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = mma(TL::col_frag(vt, cbase, wk * KT + 32 * s + 16 * t, d), p, o[d]);
            }
    };

    const int plain = mask || a.tail || end < begin ? begin : begin + (end - begin) / BN * BN;  // tiles before are whole
    int stage = 0;
    const auto steps = [&](int from, int to, auto edge) {
        for (int n0 = from; n0 < to; n0 += BN) {
            dma_wait();
            __syncthreads();  // this tile is there, and nobody reads the other one any more
            if (STAGES == 2 && n0 + BN < end) {
                fetch(n0 + BN, stage ^ 1);
                look(n0 + 2 * BN);
            }
            step(n0, stage, edge);
            if (STAGES == 2) {
                stage ^= 1;
            } else if (n0 + BN < end) {
                __syncthreads();
                fetch(n0 + BN, 0);
                look(n0 + 2 * BN);
            }
        }
    };
    steps(begin, plain, std::false_type());
    steps(plain, end, std::true_type());
    l = sum_both_halves(l);
    // A masked key starts at -inf and has zeros for features, which a query that is not finite turns into NaN: where no key of
    // this piece counts the row has seen nothing all the same.
    if (mask && __any(l != l)) {
        bool some = false;
        for (int j = begin + lane; j < end; j += 64)
            some = some || mask[j];
        if (!__any(some))
            m = NEG_INF, l = 0.0f;
    }

    if constexpr (WK > 1) {  // join the waves' pieces of the key range, in wave order
        constexpr int PIECE = 64 * 16 * DT + 128;
        static_assert((WK - 1) * WM * PIECE * 4 <= STAGES * 2 * TILE_B, "the join uses the tiles' memory");
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
    const long rid = ((long)at.b * rw.M + at.i) * ((long)rw.Hk * rw.G) + at.h;
    if (!at.valid)
        m = NEG_INF, l = 0.0f;
    if (a.po) {
        const long slot = (long)(a.slot0 + split) * a.slot_rows + rid;
        if (half == 0 && at.exists)
            a.pml[slot] = make_float2(m, l);
        // (a piece without weights is never read)
        store_column<float, DT>(a.po + slot * rw.D, o, rw.D, half, at.exists && l != 0.0f, [](float x) { return x; });
        return;
    }
    const bool none = l == 0.0f;
    if (half == 0 && at.exists)
        a.lse[((long)at.b * rw.Hk * rw.G + at.h) * rw.M + at.i] = none ? NEG_INF : (m + log2_(l)) * 0.693147180559945f;
    const float inv = none ? 0.0f : 1.0f / l;
    store_column<T, DT>((T *)a.o + at.b * a.ob + at.i * a.orow + at.h * a.oh, o, rw.D, half, at.exists,
                        [=](float x) { return none ? 0.0f : x * inv; });
}

template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (attend_fwd_per_cu(sizeof(T), DT, WM))) void attend_fwd_kernel(AttendFwd a)
{
    __shared__ __attribute__((aligned(1024))) char lds[attend_fwd_lds(sizeof(T), DT, WM, 2)];
    __shared__ __attribute__((aligned(16))) float bias[2 * attend_fwd_bn(sizeof(T), DT, WM)];
    attend_fwd_block<T, DT, WM, 2>(a, lds, bias, blockIdx.x, gridDim.x);
}

// Both parts of a shared call in one launch (two launches: 64 members over 131072 entries 242 us, one: 220).  The own part has few
// rows per workgroup whatever the first has.  That case now: 204 us = 3.5 TB/s and 675 TFLOP/s at once, 0.75 of either's rate.
template <typename T, int DT>
constexpr int own_wm() { return attend_least_wm(sizeof(T), DT); }
template <typename T, int DT, int WM>
__global__ __launch_bounds__(256, (attend_fwd_per_cu(sizeof(T), DT, WM))) void attend_pair_kernel(AttendPair a)
{
    constexpr int OWN = own_wm<T, DT>();
    constexpr int A = attend_fwd_lds(sizeof(T), DT, WM, 2), B = attend_fwd_lds(sizeof(T), DT, OWN, 1);
    constexpr int NA = 2 * attend_fwd_bn(sizeof(T), DT, WM), NB = attend_fwd_bn(sizeof(T), DT, OWN);
    __shared__ __attribute__((aligned(1024))) char lds[A > B ? A : B];
    __shared__ __attribute__((aligned(16))) float bias[NA > NB ? NA : NB];
    const unsigned n = a.first.mtiles * a.first.splits * a.first.rows.Hk;  // (one grid entry)
    if (blockIdx.x < n)
        attend_fwd_block<T, DT, WM, 2>(a.first, lds, bias, blockIdx.x, n);
    else
        attend_fwd_block<T, DT, OWN, 1>(a.second, lds, bias, blockIdx.x - n, gridDim.x - n);
}

// One wave per row: the pieces' maxima and sums (a lane each, 64 at a time), then the pieces' sums weighted by them, the two halves
// of the wave taking every other piece, four values a lane and four pieces in flight (384 rows x 21 pieces of 128: 4.4 us; one
// piece at a time: 14 us).
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendJoin a)
{
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const long rid = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rid >= a.slot_rows)
        return;
    const int d = 4 * (lane & 31);  // D is at most 128
    const float *po = a.po + rid * a.D + (d < a.D ? d : 0);
    const long step = a.slot_rows * a.D;
    float top = NEG_INF, l = 0.0f;
    f32x4 x = {0, 0, 0, 0};
    for (int s0 = 0; s0 < a.slots; s0 += 64) {
        float2 ml = make_float2(NEG_INF, 0.0f);
        if (s0 + lane < a.slots)
            ml = a.pml[(s0 + lane) * a.slot_rows + rid];
        float mn = ml.x;
#pragma unroll
        for (int k = 32; k; k >>= 1)
            mn = fmaxf(mn, __shfl_xor(mn, k));
        mn = fmaxf(mn, top);
        const float f = top == NEG_INF ? 0.0f : exp2_(top - mn);
        top = mn;
        const float w = ml.y == 0.0f ? 0.0f : exp2_(ml.x - mn);
        l = l * f + w * ml.y;
        x *= f;
        const int k = min(64, a.slots - s0);
        for (int s = 0; s < k; s += 8) {
            f32x4 p[4];
            float ws[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int mine = s + 2 * y + half, in = min(mine, k - 1);
                p[y] = *reinterpret_cast<const f32x4 *>(po + (s0 + in) * step);
                ws[y] = __shfl(w, in);
                ws[y] = mine < k ? ws[y] : 0.0f;
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x[j] += ws[y] == 0.0f ? 0.0f : ws[y] * p[y][j];  // what a piece without weights has there was never written
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1)
        l += __shfl_xor(l, k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        x[j] = sum_both_halves(x[j]);
    const int h = (int)(rid % a.H);
    const long n = rid / a.H;
    const int i = (int)(n % a.M);
    const long b = n / a.M;
    const bool none = l == 0.0f;
    if (lane == 0)
        a.lse[(b * a.H + h) * a.M + i] = none ? NEG_INF : (top + log2_(l)) * 0.693147180559945f;
    if (half == 0 && d < a.D) {
        const float inv = none ? 0.0f : 1.0f / l;
        x4<T> w;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = none ? (T)0.0f : (T)(x[j] * inv);
        *reinterpret_cast<x4<T> *>((T *)a.o + b * a.ob + i * a.orow + h * a.oh + d) = w;
    }
}

template <typename T, int DT>
void launch_fwd_dim(const AttendFwd &a, hipStream_t st)
{
    const dim3 grid((unsigned)a.blocks()), block(256);
    switch (a.wm) {
    case 1:
        if constexpr (own_wm<T, DT>() == 1)
            hipLaunchKernelGGL((attend_fwd_kernel<T, DT, 1>), grid, block, 0, st, a);
        break;
    case 2: hipLaunchKernelGGL((attend_fwd_kernel<T, DT, 2>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((attend_fwd_kernel<T, DT, 4>), grid, block, 0, st, a); break;
    }
}
template <typename T, int DT>
void launch_pair_dim(const AttendPair &a, hipStream_t st)
{
    const dim3 grid((unsigned)(a.first.blocks() + a.second.blocks())), block(256);
    switch (a.first.wm) {
    case 1:
        if constexpr (own_wm<T, DT>() == 1)
            hipLaunchKernelGGL((attend_pair_kernel<T, DT, 1>), grid, block, 0, st, a);
        break;
    case 2: hipLaunchKernelGGL((attend_pair_kernel<T, DT, 2>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((attend_pair_kernel<T, DT, 4>), grid, block, 0, st, a); break;
    }
}

}  // namespace attend

template <typename T>
void attend_launch_fwd(const AttendFwd &a, hipStream_t st)
{
    switch (attend_dt(a.rows.D)) {
    case 1: return attend::launch_fwd_dim<T, 1>(a, st);
    case 2: return attend::launch_fwd_dim<T, 2>(a, st);
    case 3: return attend::launch_fwd_dim<T, 3>(a, st);
    default: return attend::launch_fwd_dim<T, 4>(a, st);
    }
}
template <typename T>
void attend_launch_pair(const AttendPair &a, hipStream_t st)
{
    switch (attend_dt(a.first.rows.D)) {
    case 1: return attend::launch_pair_dim<T, 1>(a, st);
    case 2: return attend::launch_pair_dim<T, 2>(a, st);
    case 3: return attend::launch_pair_dim<T, 3>(a, st);
    default: return attend::launch_pair_dim<T, 4>(a, st);
    }
}
template <typename T>
void attend_launch_join(const AttendJoin &a, hipStream_t st)
{
    hipLaunchKernelGGL((attend::attend_join_kernel<T>), dim3((unsigned)((a.slot_rows + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace gpx
