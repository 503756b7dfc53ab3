// gpx_attend_tile.hpp -- fragments, LDS tiles and the matrix step shared by the attention kernels (gfx950, wave64).
//
// Everything is built from one 32 x 32 matrix step with 16 terms of the sum.  Its operand of a lane is 8 values: row (or column)
// lane % 32, terms 8 (lane / 32) .. + 7; its result is 16 values: column lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4.
// 16-bit types: one v_mfma_f32_32x32x16.  fp32: each value is cut into three bf16 pieces of 8 bits, exactly (24 bits in all), and
// six of the nine products of pieces are summed in fp32, smallest first.  The pieces of one side are cut off (every m and l has the
// sign of its value), those of the other rounded to nearest, so what the three left out add up to -- at most 3 x 2^-24 of the product:
// 2^-7 2^-17 + 2^-15 2^-8 -- has no sign of its own.  (Both cut off: 2^-21, always towards zero, so that it adds up along the
// features.  Both rounded: 2^-24, but 24 % slower, for the rounding of what the loops read.)  Measured error against 64 bits 0.4-1.0 of a
// plain fp32 form's, at 6 x 32 cycles a step where v_mfma_f32_32x32x2_f32 takes 8 x 64: 17 x 5 rows over 16384 entries 72 -> 55 us;
// 4096 x 8192, 8 heads of 128: 154 TFLOP/s, of 64: 142 (the fp32 matrix instructions' peak is 157, the library's fp32 product reaches
// 153; six products at bf16's rate are 178).  Values that are not finite become NaN.
//
// That freedom is used once more: a result tile W (rows = terms of the NEXT product) goes into it as an operand without
// leaving its lane -- registers 8 t .. 8 t + 7 are the terms { 16 t + 8 (j / 4) + 4 (lane / 32) + j % 4 } -- and the other
// operand is read from LDS in that order (col_frag).  So the weights never pass through LDS.
#pragma once
#include "gpx_attend.hpp"

namespace gpx {
namespace attend {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<float> {
    typedef float x8 __attribute__((ext_vector_type(8)));
    typedef float x4 __attribute__((ext_vector_type(4)));
};
template <> struct Elem<_Float16> {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x4 __attribute__((ext_vector_type(4)));
};
template <> struct Elem<__bf16> {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x4 __attribute__((ext_vector_type(4)));
};
template <typename T> using x8 = typename Elem<T>::x8;
template <typename T> using x4 = typename Elem<T>::x4;

// A lane's 8 values of an operand, as the matrix cores take them.
template <typename T>
struct Frag {
    x8<T> v;
    __device__ __forceinline__ static Frag of(x8<T> x) { return {x}; }
    __device__ __forceinline__ static Frag rounded(x8<T> x) { return {x}; }
    __device__ __forceinline__ float operator[](int j) const { return (float)v[j]; }
};
template <>
struct Frag<float> {
    x8<__bf16> h, m, l;  // the upper, middle and lower 8 bits of each value; their sum is the value
    // cut off: 0 <= m < 2^-7 and 0 <= l < 2^-15 of the value's size, for what the loops read (11 instructions a pair)
    __device__ __forceinline__ static Frag of(x8<float> x)
    {
        u32x4 h, m, l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = x[2 * j], b = x[2 * j + 1];
            h[j] = uppers(a, b);
            less(a, b, bits(a), bits(b));
            m[j] = uppers(a, b);
            less(a, b, bits(a), bits(b));
            l[j] = uppers(a, b);
        }
        return {__builtin_bit_cast(x8<__bf16>, h), __builtin_bit_cast(x8<__bf16>, m), __builtin_bit_cast(x8<__bf16>, l)};
    }
    // rounded to nearest: |m| <= 2^-8, |l| <= 2^-17, of either sign, for the other side: rows a wave keeps, weights, dS
    __device__ __forceinline__ static Frag rounded(x8<float> x)
    {
        constexpr float MOST = 0x1.fep127f;  // bf16's largest: what is above would round to infinity (the lower pieces hold the rest)
        u32x4 h, m, l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = x[2 * j], b = x[2 * j + 1];
            h[j] = nearest(__builtin_amdgcn_fmed3f(a, -MOST, MOST), __builtin_amdgcn_fmed3f(b, -MOST, MOST));
            less(a, b, h[j] << 16, h[j]);
            m[j] = nearest(a, b);
            less(a, b, m[j] << 16, m[j]);
            l[j] = uppers(a, b);
        }
        return {__builtin_bit_cast(x8<__bf16>, h), __builtin_bit_cast(x8<__bf16>, m), __builtin_bit_cast(x8<__bf16>, l)};
    }
    __device__ __forceinline__ static unsigned bits(float x) { return __builtin_bit_cast(unsigned, x); }
    __device__ __forceinline__ static unsigned uppers(float a, float b) { return __builtin_amdgcn_perm(bits(b), bits(a), 0x07060302); }
    __device__ __forceinline__ static unsigned nearest(float a, float b)
    {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, pair{(__bf16)a, (__bf16)b});
    }
    __device__ __forceinline__ static void less(float &a, float &b, unsigned pa, unsigned pb)  // the pieces' upper halves
    {
        a -= __builtin_bit_cast(float, pa & 0xffff0000u);
        b -= __builtin_bit_cast(float, pb & 0xffff0000u);
    }
    __device__ __forceinline__ float operator[](int j) const { return ((float)l[j] + (float)m[j]) + (float)h[j]; }
};

__device__ __forceinline__ f32x16 mma16(x8<_Float16> a, x8<_Float16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma16(x8<__bf16> a, x8<__bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
template <typename T>
__device__ __forceinline__ f32x16 mma(const Frag<T> &a, const Frag<T> &b, f32x16 c)
{
    if constexpr (sizeof(T) == 2) {
        return mma16(a.v, b.v, c);
    } else {
        c = mma16(a.l, b.h, c);
        c = mma16(a.h, b.l, c);
        c = mma16(a.m, b.m, c);
        c = mma16(a.m, b.h, c);
        c = mma16(a.h, b.m, c);
        return mma16(a.h, b.h, c);
    }
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32, 1 ulp
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }   // v_log_f32, 1 ulp
constexpr float NEG_INF = -__builtin_huge_valf(), POS_INF = __builtin_huge_valf();

// lanes l and l ^ 32 hold the two halves of every column
__device__ __forceinline__ void both_halves(float x, float &a, float &b)  // a: the lower lanes' value, b: the upper lanes'
{
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned lo = r[0], hi = r[1];  // (a bit cast of an element of a vector is one of its first element)
    a = __builtin_bit_cast(float, lo), b = __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float max_both_halves(float x)
{
    float a, b;
    both_halves(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_both_halves(float x)
{
    float a, b;
    both_halves(x, a, b);
    return a + b;
}

// 8 values of a result tile as an operand, rounded to the element type (to nearest even; fp32: pieces rounded to nearest)
template <typename T>
__device__ __forceinline__ Frag<T> as_operand(const f32x16 &w, int t)
{
    x8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        r[j] = (T)w[8 * t + j];
    return Frag<T>::rounded(r);
}

// A tile of rows of DP = 32 DT features in LDS: 16-byte chunks, LC (a power of two) per row, chunk c of row r at place
// c ^ swz(r).  swz is linear over the bits of r and chosen so that both ways of reading spread over the 64 banks: 16 rows
// at one chunk (row_frag), and 4 consecutive rows at 4 consecutive chunks (col_frag of the 16-bit types).
template <typename T, int DT>
struct Tile {
    static constexpr int ESZ = sizeof(T);
    static constexpr int EPC = 16 / ESZ;           // elements per chunk
    static constexpr int NCH = 32 * DT / EPC;      // chunks a row has
    static constexpr int ROWB = attend_row_bytes(ESZ, DT);
    static constexpr int LC = ROWB / 16;           // places a row has, a power of two
    static constexpr int KS = 2 * DT;              // matrix steps over the features

    static __device__ __host__ constexpr int swz(int r)
    {
        return LC >= 16 ? (((r & 3) << 2) | ((r >> 2) & 3)) : LC == 8 ? ((((r >> 1) & 1) << 2) | ((r >> 2) & 3)) : ((r >> 2) & 3);
    }

    // lane part of row_frag's address: row lane % 32, the lane's half of the 16 features of a step
    static __device__ __forceinline__ int row_base(int lane)
    {
        const int r = lane & 31, h = lane >> 5;
        const int c = ESZ == 2 ? h : 2 * h;
        return r * ROWB + ((c ^ swz(r)) << 4);
    }
    // rows row0 .. row0 + 31 (row0: a multiple of 32), features 16 t .. 16 t + 15
    static __device__ __forceinline__ Frag<T> row_frag(const char *tile, int base, int row0, int t)
    {
        if constexpr (ESZ == 2) {
            return Frag<T>::of(__builtin_bit_cast(x8<T>, *reinterpret_cast<const u32x4 *>(tile + row0 * ROWB + (base ^ (t << 5)))));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(tile + row0 * ROWB + (base ^ (t << 6)));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(tile + row0 * ROWB + (base ^ (t << 6) ^ 16));
            return Frag<T>::of(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    // lane part of col_frag's address.  16-bit: ds_read_b64_tr_b16 takes from each lane of a block of 16 the address of 4
    // values, 4 lanes to a row, and hands lane i column i of that 4 x 16 block.
    static __device__ __forceinline__ int col_base(int lane)
    {
        const int h = lane >> 5;
        if constexpr (ESZ == 2) {
            const int i = lane & 15, blk = (lane >> 4) & 1;
            const int row = 4 * h + (i >> 2), c = 2 * blk + ((i & 3) >> 1);
            return row * ROWB + ((c ^ swz(row)) << 4) + ((i & 1) << 3);
        } else {
            const int d = lane & 31, row = 4 * h;
            return row * ROWB + (((d >> 2) ^ swz(row)) << 4) + ((d & 3) << 2);
        }
    }
    // column 32 dt + lane % 32 of the rows row0 + { 8 (j / 4) + 4 (lane / 32) + j % 4 }, j = 0 .. 7 (row0: a multiple of 16)
    static __device__ __forceinline__ Frag<T> col_frag(const char *tile, int base, int row0, int dt)
    {
        if constexpr (ESZ == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const char *p0 = tile + row0 * ROWB + (base ^ (dt << 6));
            const char *p1 = tile + (row0 + 8) * ROWB + (base ^ (dt << 6) ^ (swz(8) << 4));
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p0);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p1);
            return Frag<T>::of(__builtin_bit_cast(x8<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
        } else {
            x8<T> r;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = 8 * (j >> 2) + (j & 3);
                r[j] = *reinterpret_cast<const float *>(tile + (row0 + k) * ROWB + (base ^ (dt << 7) ^ (swz(k) << 4)));
            }
            return Frag<T>::of(r);
        }
    }
};

// Where a packed row's query lives (AttendRows): batch entry, query and head.
struct RowAt {
    int b, i, h;
    bool valid;  // the row exists and counts
    bool exists;
};
__device__ __forceinline__ RowAt row_at(const AttendRows &rw, int bz, int hk, int r)
{
    RowAt w;
    const int n = rw.by_g(r), g = r - n * rw.G;
    const int db = rw.by_m(n);
    w.b = bz + db;
    w.i = n - db * rw.M;
    w.h = hk * rw.G + g;
    w.exists = r < rw.R;
    w.valid = w.exists;
    if (rw.len && w.exists)
        w.valid = w.i < rw.len[w.b];
    return w;
}

// operand fragments of one row per lane straight from memory (zero where the row does not count or the feature is padding)
template <typename T, int DT>
__device__ __forceinline__ void load_row_frags(Frag<T> (&f)[2 * DT], const T *p, bool valid, int D, int lane)
{
    const int h = lane >> 5;
#pragma unroll
    for (int t = 0; t < 2 * DT; ++t) {
        const int d = 16 * t + 8 * h;
        x8<T> z;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            z[j] = (T)0.0f;
        if (valid && d < D) {
            if constexpr (sizeof(T) == 4)  // (16-byte boundaries, not 32)
                z = __builtin_shufflevector(*reinterpret_cast<const f32x4 *>(p + d), *reinterpret_cast<const f32x4 *>(p + d + 4), 0, 1, 2, 3, 4, 5, 6, 7);
            else
                z = *reinterpret_cast<const x8<T> *>(p + d);
        }
        f[t] = Frag<T>::rounded(z);
    }
}

__device__ __forceinline__ int clamped(const int *len, int b, int n)
{
    if (!len)
        return n;
    const int l = len[b];
    return l < 0 ? 0 : (l > n ? n : l);
}

// Consecutive workgroups go round the 8 XCDs, and each XCD has an L2 of its own.  Workgroup -> (tile, group), the tiles of a group
// reading the same keys (or rows): ATTEND_WHOLE_GROUPS gives XCD x the groups x, x + 8, .. with all their tiles, ATTEND_PIECES a
// contiguous piece of the list of all tiles, ATTEND_SPREAD every eighth tile.  (Pieces gave each of eight ragged objects an XCD of
// its own, which then waited for the largest: 49 us, whole heads spread over the XCDs 38.)
__device__ __forceinline__ void place_block(unsigned id, unsigned total, int order, int tiles, const DivBy &by_tiles, int &tile, int &group)
{
    unsigned at = id;
    if (order != ATTEND_SPREAD)
        at = id >> 3;
    if (order == ATTEND_PIECES) {
        const unsigned per = total >> 3, rest = total & 7, x = id & 7;
        at += x * per + (x < rest ? x : rest);
    }
    const int u = by_tiles(at);
    tile = at - u * tiles;
    group = order == ATTEND_WHOLE_GROUPS ? u * 8 + (int)(id & 7) : u;
}

// The batch entry of the p-th longest key range, for batches of up to 64 that take more than one round of workgroups: the longest
// ranges are started first, so that a ragged batch does not end on one of them (nine clouds, 2841 queries each: 45.6 -> 40.6 us;
// where all workgroups run at once the sorting only costs its half microsecond).  Which workgroup does what changes no result.
__device__ __forceinline__ int nth_longest(const AttendKeys &keys, int batch, int p)
{
    if (!keys.sort)
        return p;
    const int lane = threadIdx.x & 63;
    const int mine = lane < batch ? clamped(keys.len, lane, keys.n) : -1;
    int rank = 0;
    for (int j = 0; j < batch; ++j) {
        const int other = __builtin_amdgcn_readlane(mine, j);
        rank += other > mine || (other == mine && j < lane);
    }
    return __builtin_ctzll(__ballot(lane < batch && rank == p));
}

// ---- memory -> LDS without registers -------------------------------------------------------------------------------------------
// buffer_load_dwordx4 .. lds: lane i's 16 bytes land at M0 + 16 i, so one instruction fills 64 consecutive places of a tile and the
// lanes choose which chunk goes where by their addresses (the swizzle of Tile).  Offsets are 32 bits relative to a 64-bit base
// that moves with the tile; an offset outside the buffer delivers zeros, which is how rows past the end, rows that do not count
// and padding features become zeros.  The compiler does not see these loads: dma_wait() comes before the barrier behind which a
// tile is read.  M0 is reserved (never allocated; what the compiler uses it for, it sets right before), so it is no clobber.
constexpr unsigned DMA_OUT = 0x80000000u;    // an offset that is outside every buffer
constexpr unsigned DMA_MOST = 0x7fffffffu;   // bytes a buffer has at most

__device__ __forceinline__ u32x4 dma_buffer(const void *base, unsigned bytes)
{
    const unsigned long long p = (unsigned long long)base;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((unsigned)p);
    r[1] = __builtin_amdgcn_readfirstlane((unsigned)(p >> 32)) & 0xffffu;
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000u;
    return r;
}
__device__ __forceinline__ void dma16(u32x4 buffer, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}
__device__ __forceinline__ void dma4(u32x4 buffer, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}
// (the builtin tells the compiler that its own loads have arrived too: without it, fragments loaded before a loop are waited for at
// their first use inside it, in every round, and with them the tile that was just asked for)
__device__ __forceinline__ void dma_wait()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
}
__device__ __forceinline__ unsigned lds_offset(const void *p) { return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char *)p; }

// how the 4 waves of a workgroup fill a tile of BN rows: instruction x of a wave takes the places from 64 (4 x + wave) on
template <typename T, int DT, int BN>
struct Fill {
    using TL = Tile<T, DT>;
    static constexpr int WI = BN * TL::LC / 64;  // instructions of the tile
    static constexpr int N = (WI + 3) / 4;       // of a wave
    static constexpr int RPI = 64 / TL::LC;      // rows of an instruction
    static_assert(BN * TL::LC % 64 == 0, "whole instructions");

    static __device__ __forceinline__ bool on(int x, int wave) { return WI % 4 == 0 || 4 * x + wave < WI; }
    static __device__ __forceinline__ int row(int x, int wave, int lane) { return (4 * x + wave) * RPI + lane / TL::LC; }
    // the lane's chunk as a byte offset in its row; DMA_OUT where it is padding
    static __device__ __forceinline__ unsigned chunk(int x, int wave, int lane, int D)
    {
        const int c = (lane % TL::LC) ^ TL::swz(row(x, wave, lane));
        return c * TL::EPC < D ? 16u * c : DMA_OUT;
    }
    static __device__ __forceinline__ unsigned lds(int x, int wave) { return 1024u * (4 * x + wave); }
};

// A lane's column of a result of DT tiles (rows = features) to memory, rounded once: f(value) -> value to store.  A lane holds 4
// consecutive features at a time, the other half of the wave the next 4; the 16-bit types swap pieces between the halves first,
// so that every store is 16 bytes.  Features from D on are padding.
template <typename T, int DT, typename F>
__device__ __forceinline__ void store_column(T *p, const f32x16 (&r)[DT], int D, int half, bool on, F f)
{
    if constexpr (sizeof(T) == 4) {
        if (!on)
            return;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int at = 32 * d + 8 * x + 4 * half;
                if (at < D)
                    *reinterpret_cast<f32x4 *>(p + at) = f32x4{f(r[d][4 * x]), f(r[d][4 * x + 1]), f(r[d][4 * x + 2]), f(r[d][4 * x + 3])};
            }
    } else {
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
                x4<T> a, b;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[j] = (T)f(r[d][4 * x + j]);
                    b[j] = (T)f(r[d][4 * x + 4 + j]);
                }
                u32x2 ua = __builtin_bit_cast(u32x2, a), ub = __builtin_bit_cast(u32x2, b);
                unsigned a0 = ua[0], a1 = ua[1], b0 = ub[0], b1 = ub[1];
                // the upper lanes' a for the lower lanes' b: then a lane has 8 features in a row, of piece x or x + 1
                asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %2\n\tv_permlane32_swap_b32 %1, %3" : "+v"(a0), "+v"(a1), "+v"(b0), "+v"(b1));
                const int at = 32 * d + 8 * (x + half);
                if (on && at < D)
                    *reinterpret_cast<u32x4 *>(p + at) = u32x4{a0, a1, b0, b1};
            }
    }
}

// weights of masked places: register i of a result tile is row 8 (i / 4) + 4 half + i % 4
__device__ __forceinline__ bool bit_of(unsigned m, int half, int i) { return (m >> (8 * (i >> 2) + 4 * half + (i & 3))) & 1u; }

}  // namespace attend
}  // namespace gpx
