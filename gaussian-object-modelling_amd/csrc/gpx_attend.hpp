// gpx_attend.hpp -- softmax-weighted sums over a context (gpx_attend, gpx_attend_backward, gpx_attend_shared of include/gpx.h):
// what the host side (gpx_attend.hip) hands to the kernels, and the launchers of the three element types.
#pragma once
#include "gpx_internal.hpp"

namespace gpx {

constexpr int ATTEND_MAX_DIM = 128;
constexpr double ATTEND_LOG2E = 1.4426950408889634074;

// One set of keys and values: element strides of batch, row and head.
struct AttendKeys {
    const void *k = nullptr, *v = nullptr;
    long kb = 0, kr = 0, kh = 0, vb = 0, vr = 0, vh = 0;
    int n = 0;                        // rows the tensors have
    const int *len = nullptr;         // rows that count per batch entry (clamped to [0, n]); null: n
    const unsigned char *mask = nullptr;  // nonzero: the row counts; [batch][mask_b]; null: all
    long mask_b = 0;
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
};

struct AttendFwd {
    AttendRows rows;
    AttendKeys keys;
    float c = 0;            // scale log2(e): weights are 2^(c s - m)
    int tail = 0;           // 1: query i sees keys < len - (M - 1 - i)
    int splits = 1, chunk = 0;  // the key range in pieces of `chunk` rows, one workgroup each
    void *o = nullptr;      // splits == 1 and po == null
    long ob = 0, orow = 0, oh = 0;
    float *lse = nullptr;   // [B][H][M]
    float *po = nullptr;    // else: unnormalised sums [slot][rid][D], rid = ((b M + i) H + h)
    float2 *pml = nullptr;  // and their maximum (log2 units) and sum of weights [slot][rid]
    int slot0 = 0;
    long slot_rows = 0;
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

struct AttendBwd {
    AttendRows rows;
    AttendKeys keys;
    float c = 0, scale = 0;
    const void *o = nullptr, *dout = nullptr;
    long ob = 0, orow = 0, oh = 0, gb = 0, gr = 0, gh = 0;
    const float *lse = nullptr;
    float *stat = nullptr;   // [2][B][H][M]: lse in log2 units (+inf where the row has no weights); <dO, O>
    DivBy div_g;             // by rows.G
    void *dq = nullptr, *dk = nullptr, *dv = nullptr;
    long dqb = 0, dqr = 0, dqh = 0, dkb = 0, dkr = 0, dkh = 0, dvb = 0, dvr = 0, dvh = 0;
    int q_splits = 1, q_chunk = 0;   // dQ: pieces of the key range
    int k_splits = 1, k_chunk = 0;   // dK, dV: pieces of the row range
    float *pq = nullptr;             // q_splits > 1: partial dQ [split][rid][D]
    float *pk = nullptr, *pv = nullptr;  // k_splits > 1: [split][(b Hk + hk) n + j][D]
};

// rows of the packed enumeration one workgroup takes / keys it takes per step, by the number of rows and the element type
int attend_block_rows(bool f32, int dim, int rows);
int attend_block_keys(bool f32, int dim, int rows);
constexpr int ATTEND_DKV_KEYS = 128;  // keys of one workgroup of the dK, dV kernel
int attend_dkv_block_rows(bool f32);

template <typename T> void attend_launch_fwd(const AttendFwd &a, hipStream_t st);
template <typename T> void attend_launch_join(const AttendJoin &a, hipStream_t st);
template <typename T> void attend_launch_bwd(const AttendBwd &a, hipStream_t st);

}  // namespace gpx
