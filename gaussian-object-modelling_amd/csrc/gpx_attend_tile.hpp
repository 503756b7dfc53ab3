// gpx_attend_tile.hpp -- fragments, LDS tiles and the matrix step shared by the attention kernels (gfx950, wave64).
//
// Everything is built from one 32 x 32 matrix step with 16 terms of the sum.  Its operand of a lane is 8 values: row (or column)
// lane % 32, terms 8 (lane / 32) .. + 7; its result is 16 values: column lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4.
// 16-bit types: one v_mfma_f32_32x32x16; fp32: eight v_mfma_f32_32x32x2 over the same 8 values (the order of the terms does
// not matter as long as both operands agree on it).
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

__device__ __forceinline__ f32x16 mma(x8<_Float16> a, x8<_Float16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(x8<__bf16> a, x8<__bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(x8<float> a, x8<float> b, f32x16 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32, 1 ulp
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }   // v_log_f32, 1 ulp
constexpr float NEG_INF = -__builtin_huge_valf(), POS_INF = __builtin_huge_valf();

// lanes l and l ^ 32 hold the two halves of every column
__device__ __forceinline__ void both_halves(float x, float &a, float &b)  // a: the lower lanes' value, b: the upper lanes'
{
    unsigned u = __builtin_bit_cast(unsigned, x), w = u;
    // (the builtin hands back its first result twice; two wait states after the instruction that wrote an operand)
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(u), "+v"(w));
    a = __builtin_bit_cast(float, u), b = __builtin_bit_cast(float, w);
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

// 8 values of a result tile as an operand, rounded to the element type (to nearest even; fp32: kept)
template <typename T>
__device__ __forceinline__ x8<T> as_operand(const f32x16 &w, int t)
{
    x8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        r[j] = (T)w[8 * t + j];
    return r;
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
    static __device__ __forceinline__ int place(int row, int chunk) { return row * ROWB + ((chunk ^ swz(row)) << 4); }

    // lane part of row_frag's address: row lane % 32, the lane's half of the 16 features of a step
    static __device__ __forceinline__ int row_base(int lane)
    {
        const int r = lane & 31, h = lane >> 5;
        const int c = ESZ == 2 ? h : 2 * h;
        return r * ROWB + ((c ^ swz(r)) << 4);
    }
    // rows row0 .. row0 + 31 (row0: a multiple of 32), features 16 t .. 16 t + 15
    static __device__ __forceinline__ x8<T> row_frag(const char *tile, int base, int row0, int t)
    {
        if constexpr (ESZ == 2) {
            return __builtin_bit_cast(x8<T>, *reinterpret_cast<const u32x4 *>(tile + row0 * ROWB + (base ^ (t << 5))));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(tile + row0 * ROWB + (base ^ (t << 6)));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(tile + row0 * ROWB + (base ^ (t << 6) ^ 16));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
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
    static __device__ __forceinline__ x8<T> col_frag(const char *tile, int base, int row0, int dt)
    {
        if constexpr (ESZ == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const char *p0 = tile + row0 * ROWB + (base ^ (dt << 6));
            const char *p1 = tile + (row0 + 8) * ROWB + (base ^ (dt << 6) ^ (swz(8) << 4));
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p0);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p1);
            return __builtin_bit_cast(x8<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            x8<T> r;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = 8 * (j >> 2) + (j & 3);
                r[j] = *reinterpret_cast<const float *>(tile + (row0 + k) * ROWB + (base ^ (dt << 7) ^ (swz(k) << 4)));
            }
            return r;
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
__device__ __forceinline__ void load_row_frags(x8<T> (&f)[2 * DT], const T *p, bool valid, int D, int lane)
{
    const int h = lane >> 5;
#pragma unroll
    for (int t = 0; t < 2 * DT; ++t) {
        const int d = 16 * t + 8 * h;
        x8<T> z;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            z[j] = (T)0.0f;
        f[t] = z;
        if (valid && d < D)
            f[t] = *reinterpret_cast<const x8<T> *>(p + d);
    }
}

__device__ __forceinline__ int clamped(const int *len, int b, int n)
{
    if (!len)
        return n;
    const int l = len[b];
    return l < 0 ? 0 : (l > n ? n : l);
}

// Consecutive workgroups go round the 8 XCDs: give each XCD a contiguous piece of the work, so that workgroups that read
// the same keys share an L2.
__device__ __forceinline__ unsigned xcd_order(unsigned id, unsigned total)
{
    const unsigned per = total >> 3, rest = total & 7, x = id & 7, at = id >> 3;
    return x * per + (x < rest ? x : rest) + at;
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

// weights of masked places: register i of a result tile is row 8 (i / 4) + 4 half + i % 4
__device__ __forceinline__ bool bit_of(unsigned m, int half, int i) { return (m >> (8 * (i >> 2) + 4 * half + (i & 3))) & 1u; }

}  // namespace attend
}  // namespace gpx
