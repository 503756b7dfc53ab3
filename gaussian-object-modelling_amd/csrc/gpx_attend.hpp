// gpx_attend.hpp -- softmax-weighted sums over a context (gpx_attend, gpx_attend_backward, gpx_attend_shared of include/gpx.h):
// what the host side (gpx_attend.hip) hands to the kernels, and the launchers of the three element types.
#pragma once
#include "gpx_internal.hpp"

namespace gpx {

constexpr int ATTEND_MAX_DIM = 128;
constexpr double ATTEND_LOG2E = 1.4426950408889634074;

// n / d for 0 <= n < 2^31 by a product (d >= 1): with 2^s >= d and f = floor(2^32 (2^s - d) / d) + 1 the quotient is
// floor((n + floor(n f / 2^32)) / 2^s)
struct DivBy {
    unsigned f = 1, s = 0;
    DivBy() = default;
    explicit DivBy(unsigned d)
    {
        while ((1u << s) < d)
            ++s;
        f = (unsigned)((((unsigned long long)1 << 32) * (((unsigned long long)1 << s) - d)) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((unsigned)n, f) + (unsigned)n) >> s); }
};

// One set of keys and values: element strides of batch, row and head.
struct AttendKeys {
    const void *k = nullptr, *v = nullptr;
    long kb = 0, kr = 0, kh = 0, vb = 0, vr = 0, vh = 0;
    int n = 0;                        // rows the tensors have
    const int *len = nullptr;         // rows that count per batch entry (clamped to [0, n]); null: n
    const unsigned char *mask = nullptr;  // nonzero: the row counts; [batch][mask_b]; null: all
    long mask_b = 0;
    int sort = 0;                     // 1: the batch entries in the order of their lengths, longest first (at most 64 of them)
};

// Queries are enumerated per (grid batch entry, key head) as packed rows r = n G + g, g the head inside the group of G heads
// that share a key head and n = 0 .. rows / G - 1: batch entry bz + n / M, query n % M.  A call over a batch has n < M; the
// shared context takes all batch entries as rows of ONE grid entry.
struct AttendRows {
    const void *q = nullptr;
    long qb = 0, qr = 0, qh = 0;
    const int *len = nullptr;  // queries that count per batch entry (clamped to [0, M]); null: M
    int R = 0, M = 0, G = 1, Hk = 1, D = 0;
    int grid_b = 1;   // batch entries of the grid
    DivBy by_m, by_g, by_hk;
};

// which workgroups share an XCD (gpx_attend_tile.hpp, place_block); whole groups need a multiple of 8 of them
enum { ATTEND_WHOLE_GROUPS = 0, ATTEND_PIECES = 1, ATTEND_SPREAD = 2 };
inline int attend_order(int tiles, long groups, bool ragged)
{
    return tiles > 1 && groups % 8 == 0 ? ATTEND_WHOLE_GROUPS : tiles > 1 && ragged ? ATTEND_SPREAD : ATTEND_PIECES;
}

struct AttendFwd {
    AttendRows rows;
    AttendKeys keys;
    float c = 0;            // scale log2(e): weights are 2^(c s - m)
    int tail = 0;           // 1: query i sees keys < len - (M - 1 - i)
    int splits = 1, chunk = 0;  // the key range in pieces of `chunk` rows, one workgroup each
    int wm = 4, mtiles = 1;     // waves and workgroups along the rows
    DivBy by_mtiles, by_splits;
    int order = 0;
    void *o = nullptr;      // splits == 1 and po == null
    long ob = 0, orow = 0, oh = 0;
    float *lse = nullptr;   // [B][H][M]
    float *po = nullptr;    // else: unnormalised sums [slot][rid][D], rid = ((b M + i) H + h)
    float2 *pml = nullptr;  // what their weights are relative to (log2 units) and the sum of weights [slot][rid]
    int slot0 = 0;
    long slot_rows = 0;

    int blocks() const { return mtiles * splits * rows.Hk * rows.grid_b; }
};

// The shared context and the own part in one launch: workgroups of the first, then of the second.
struct AttendPair {
    AttendFwd first, second;
};

// Joins the pieces: o = sum_s 2^(m_s - m) po_s / l.  grid: one wave per row.
struct AttendJoin {
    const float *po = nullptr;
    const float2 *pml = nullptr;
    int slots = 0;
    long slot_rows = 0;
    int M = 0, H = 1, D = 0;
    void *o = nullptr;
    long ob = 0, orow = 0, oh = 0;
    float *lse = nullptr;
};

struct AttendBwd {
    AttendRows rows;
    AttendKeys keys;
    float c = 0, scale = 0;
    const void *o = nullptr, *dout = nullptr;
    long ob = 0, orow = 0, oh = 0, gb = 0, gr = 0, gh = 0;
    const float *lse = nullptr;
    float *stat = nullptr;   // [2][B][H][M], from the dQ kernel for the dK, dV one: lse in log2 units (+inf where the row has no
                             // weights); <dO, O>
    void *dq = nullptr, *dk = nullptr, *dv = nullptr;
    long dqb = 0, dqr = 0, dqh = 0, dkb = 0, dkr = 0, dkh = 0, dvb = 0, dvr = 0, dvh = 0;
    int fused = 0;                   // dQ and dK, dV in one launch
    int q_splits = 1, q_chunk = 0;   // dQ: pieces of the key range
    int wm = 4;                      // dQ: waves along the rows
    int mtiles = 1, ktiles = 1;      // workgroups along the rows (dQ) and along the keys (dK, dV)
    DivBy by_mtiles, by_ktiles, by_q_splits, by_k_splits;
    int q_order = 0, k_order = 0;
    int k_splits = 1, k_chunk = 0;   // dK, dV: pieces of the row range
    float *pq = nullptr;             // q_splits > 1: partial dQ [split][rid][D]
    float *pk = nullptr, *pv = nullptr;  // k_splits > 1: [split][(b Hk + hk) n + j][D]
};

// ---- tile shapes (esz: bytes of an element, dt: 32-feature pieces of a row) ---------------------------------------------------
constexpr int attend_dt(int dim) { return (dim + 31) / 32; }
constexpr int attend_row_bytes(int esz, int dt)  // of a row in LDS: a power of two
{
    int p = 64;
    while (p < 32 * dt * esz)
        p *= 2;
    return p;
}
// Waves along the rows (32 packed rows each): 1, 2 or 4; what is left of a workgroup's 4 waves takes parts of the key range.  (fp32
// rows of more than 64 features: two at least, four waves' tiles of keys would not fit.)
constexpr int attend_least_wm(int esz, int dt) { return esz == 4 && dt > 2 ? 2 : 1; }
constexpr int attend_fwd_kt(int esz, int dt, int wm) { return esz == 2 && wm == 4 ? 64 : 32; }  // keys of a wave per step
constexpr int attend_fwd_bn(int esz, int dt, int wm) { return attend_fwd_kt(esz, dt, wm) * (4 / wm); }
constexpr int attend_fwd_lds(int esz, int dt, int wm, int stages) { return stages * 2 * attend_fwd_bn(esz, dt, wm) * attend_row_bytes(esz, dt); }
constexpr int attend_lds_per_cu(int bytes) { return bytes <= 38 * 1024 ? 4 : bytes <= 52 * 1024 ? 3 : bytes <= 78 * 1024 ? 2 : 1; }
// workgroups a CU holds: LDS, and the registers of a wave (512 a SIMD lane, so waves per SIMD = workgroups per CU)
constexpr int attend_fwd_per_cu(int esz, int dt, int wm)
{
    const int regs = esz == 4 ? (dt == 1 ? 3 : dt <= 3 ? 2 : 1) : dt <= 2 ? 3 : 2;
    const int lds = attend_lds_per_cu(attend_fwd_lds(esz, dt, wm, 2));
    return lds < regs ? lds : regs;
}
constexpr int attend_dq_bn(int wm) { return 32 * (4 / wm); }
constexpr int attend_dq_lds(int esz, int dt, int wm) { return 4 * attend_dq_bn(wm) * attend_row_bytes(esz, dt); }
constexpr int attend_dq_per_cu(int esz, int dt, int wm)
{
    const int regs = esz == 4 ? (dt > 2 ? 1 : 2) : dt <= 2 ? 3 : 2;
    const int lds = attend_lds_per_cu(attend_dq_lds(esz, dt, wm));
    return lds < regs ? lds : regs;
}
constexpr int ATTEND_DKV_KEYS = 128;  // keys of one workgroup of the dK, dV kernel
constexpr int attend_dkv_br(int esz) { return esz == 2 ? 64 : 32; }
constexpr int attend_dkv_per_cu(int esz, int dt) { return esz == 2 ? (dt <= 2 ? 3 : 2) : dt <= 2 ? 2 : 1; }

constexpr int attend_dkv_lds(int esz, int dt, bool own) { return (own ? 6 : 4) * attend_dkv_br(esz) * attend_row_bytes(esz, dt); }
constexpr int attend_both_per_cu(int esz, int dt, int wm)
{
    const int q = attend_dq_per_cu(esz, dt, wm), k = attend_dkv_per_cu(esz, dt), lds = attend_lds_per_cu(attend_dkv_lds(esz, dt, true));
    const int regs = q < k ? q : k;
    return lds < regs ? lds : regs;
}

template <typename T> void attend_launch_fwd(const AttendFwd &a, hipStream_t st);
template <typename T> void attend_launch_pair(const AttendPair &a, hipStream_t st);
template <typename T> void attend_launch_join(const AttendJoin &a, hipStream_t st);
template <typename T> void attend_launch_bwd(const AttendBwd &a, hipStream_t st);

}  // namespace gpx
