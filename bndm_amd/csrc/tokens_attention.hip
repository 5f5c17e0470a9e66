// Differential attention  o = (P1 - lam P2) v,  P_m = softmax(scale q_m k_m^T), and its gradients, on the matrix units.
//
// Forward: one pass over the keys, with a running maximum and sum for each map, which are a wave's each; the scores are formed TRANSPOSED
// (keys down, queries across), so a lane holds one query: maxima and sums are over its own registers, its running statistics are
// scalars to it, and the weights of a step are at once the right operand of  o^T += v^T P^T.  v^T comes out of LDS by transposing
// reads.  For few queries the keys are split over workgroups and the parts joined by a second kernel.
//
// Backward, with dP = do v^T (the same for both maps), D_m = rowsum(P_m dP) = do . o_m:
//   dS1 = P1 (dP - D1),  dS2 = -lam P2 (dP - D2),  dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P1 - lam P2)^T do,
//   dlam = - sum over rows of D2.
// A kernel for D_m, one for the queries and one for the keys, each with the sums it owns in registers: no atomics, and the same result every
// time.
//
// Statistics, sums and gradients' sums are 32 bits.  The matrix units take products of 16-bit operands.  Where a sum cancels, its weights go there
// in two parts, as rounded and what that left off: P in the forward pass (the maps' common part), dS in dq (a row's dS adds up to 0: the keys'
// common part).  P1 - lam P2 for dv and dS for dk are rounded once, like a value that is stored.
#include "tokens_common.hpp"
#include <cmath>

namespace bndm {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLowest = -3.0e38f;
constexpr int THREADS = 256;

struct Args {
    const void *q, *k, *v, *lam;
    const int32_t *q_start, *kv_lengths;
    void *o, *o2;
    float *lse;                     // [B, 2H, Nq], log2 of the sums of exp2(scale log2(e) score); +inf for a row that sees nothing
    int64_t Nq, Nk;
    int64_t qb, qn, qh, kb, kn, kh, vb, vn, vh;
    int B, H, Hk, D, Dv;
    int causal, lam_f32;
    float scale;
    // forward
    int heads_per_row;              // query heads that share a workgroup's rows (packed after one another), 1 or H / Hk
    int splits;                     // parts of the keys
    int64_t split_keys;             // keys of a part, a multiple of the tile
    float *part;                    // [B, H, Nq, splits][2 Dv + 4]: both maps' sums, then their maxima and totals
    // backward
    const void *dout;
    int64_t dob, don, doh;
    void *dq, *dk, *dv, *dlam;
    float *delta;                   // [B, 2H, Nq]: D1, D2
    float *d2_sums;                 // [H, B, runs of 32 queries, up to a multiple of 4]: sums of D2
    float *peaks;                   // [B, H, the same runs]: the largest max(1, |lam|) |dP|
    float *steps;                   // [B, Hk]: a power of two that dS is multiplied by on its way to the matrix units
};

// Copies tiles of R rows of C chunks into LDS, NW waves together.  Rows past rows_in and chunks past the head's size become zeros.  A lane's
// offset is the same for all its pieces but for whole rows, which the scalar offset adds.
template <int R, int C, int NW, bool COLUMNS = false> struct Stager {      // COLUMNS: a tile that is only read transposed
    static constexpr int N = R * C < 64 * NW ? 1 : R * C / (64 * NW), STEP = 64 * NW / C;  // pieces of a lane, rows between them
    int row;
    uint32_t off[STEP % 16 ? 16 / STEP : 1];                // (the swizzle's period is 16 rows)
    int step_bytes;

    __device__ __forceinline__ void begin(int64_t stride, int chunks_in, int w, int l) {
        const int at = w * 64 + l;
        row = at / C;
        step_bytes = (int)stride * STEP * 2;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(off) / 4); ++i) {
            int c = at % C;
            if constexpr (COLUMNS) c ^= swizzle_columns<C>(row + i * STEP);
            else c ^= swizzle<C>(row + i * STEP);
            off[i] = c < chunks_in ? (uint32_t)(row * (int)stride + c * 8) * 2u : kNowhere;
        }
    }
    __device__ __forceinline__ void copy(char *lds, const void *base, int rows_in, int w) const {
        if (R * C < 64 * NW && w * 64 >= R * C) return;     // (fewer pieces than lanes: the first waves')
        const __amdgpu_buffer_rsrc_t rs = uniform_rsrc(base, kAnywhere);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t o = row < rows_in - i * STEP ? off[i % (sizeof(off) / 4)] : kNowhere;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (i * NW + w) * 1024), 16, o, i * step_bytes, 0, 0);
        }
    }
};

// Reads of a tile with rows of C chunks.  The swizzle is an exclusive or of a row's bits, which 32-row blocks (16 for columns) do not
// reach, so that a lane's addresses differ by constants and by constant bits of the chunk.
template <int C> struct RowReader {                    // 8 values (chunk 2 s + l / 32) of row block * 32 + l % 32
    int at;
    __device__ __forceinline__ void begin(int l) { at = (l & 31) * (C * 16) + (((l >> 5) ^ swizzle<C>(l & 31)) << 4); }
    __device__ __forceinline__ s16x8 read(const char *lds, int block, int s) const {
        return *reinterpret_cast<const s16x8 *>(lds + (at ^ ((s & 7) << 5)) + (s >> 3) * 256 + block * (32 * C * 16));
    }
};
template <int C, bool COLUMNS = false> struct ColumnReader {       // operand whose rows are the tile's COLUMNS 32 t .. + 31 and whose k are its rows
    int at;                                            // row0 .. row0 + 15 in the order in which a result tile holds them: lane half h has
    __device__ __forceinline__ void begin(int l) {     // rows row0 + 4 h + {0..3} and row0 + 8 + 4 h + {0..3}
        const int i = l & 15, col = (l & 16) + 4 * (i & 3), row = 4 * (l >> 5) + (i >> 2);
        int c = col >> 3;
        if constexpr (COLUMNS) c ^= swizzle_columns<C>(row);
        else c ^= swizzle<C>(row);
        at = row * (C * 16) + (c << 4) + (col & 4) * 2;
    }
    __device__ __forceinline__ s16x8 read(const char *lds, int row0, int t) const {
        const char *p = lds + row0 * (C * 16) + (t >> 2) * 256;
        return join(lds_read_tr(p + (at ^ ((t & 3) << 6))), lds_read_tr(p + (at ^ ((t & 3) << 6) ^ (COLUMNS ? 0 : 32)) + 8 * C * 16));
    }
};

// Workgroups go to the 8 XCDs in turn.  This deals out heads (the units that share keys, `tiles` workgroups each) to the XCDs, so that one's
// workgroups run behind one L2, and within a head the last tile first: with a causal mask it is the longest.  An XCD's second 32
// workgroups begin beside its first 32, one on each of its CUs: every other 32 go the other way, so that long ones meet short ones (the
// forward pass of 4 x 2047 causal tokens of ragged lengths and 8 heads 97 us, 114 without; the queries' gradients 73 and 81).
__device__ __forceinline__ void place(int id, int units, int tiles, int &unit, int &tile) {
    const int even = units & ~7;
    if (id < even * tiles) {
        int seq = id >> 3;
        if ((seq & 32) && (seq | 31) < even / 8 * tiles) seq ^= 31;
        unit = (seq / tiles) * 8 + (id & 7);
        tile = tiles - 1 - seq % tiles;
    } else {
        id -= even * tiles;
        unit = even + id / tiles;
        tile = tiles - 1 - id % tiles;
    }
}

// registers 8 s .. 8 s + 7 of a result tile as an operand whose k are rows 16 s .. 16 s + 15 in that order
template <typename T> __device__ __forceinline__ s16x8 as_operand(const f32x16 &p, int s) {
    return pack8<T>(p[8 * s], p[8 * s + 1], p[8 * s + 2], p[8 * s + 3], p[8 * s + 4], p[8 * s + 5], p[8 * s + 6], p[8 * s + 7]);
}

// what rounding to `p` left off them, as an operand likewise
template <typename T> __device__ __forceinline__ s16x8 rest_of(f32x16 x, const s16x8 &p, int s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { const short i = p[e]; x[8 * s + e] -= widen<T>(i); }        // (exact)
    return as_operand<T>(x, s);
}

__device__ __forceinline__ int tile_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

template <int N> __device__ __forceinline__ void clear(f32x16 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] = 0.f;
}

// of the two lanes that hold one query
__device__ __forceinline__ float both_halves_max(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t a = r.x, b = r.y;
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float both_halves_sum(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t a = r.x, b = r.y;
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// the wave's copies into LDS have landed and its reads of LDS have been answered; then every wave's
template <int NW> __device__ __forceinline__ void tile_there() {
    if constexpr (NW == 1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 32 rows of DV results, a lane's row in result-tile order, through LDS (`own`: the wave's 32 DV elements) to rows of 16-byte pieces:
// row r goes to to[offset of lane r], where `in`; f(t, r) is the value in register r of tile t.
template <typename T, int DV, typename F>
__device__ __forceinline__ void store_rows(char *own, T *to, int64_t offset, bool in, int Dv, int l, F f) {
    constexpr int C = DV / 8;
#pragma unroll
    for (int t = 0; t < DV / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int row = l & 31, col = 32 * t + tile_row(r, l >> 5);
            *reinterpret_cast<s16x4 *>(own + row * (DV * 2) + (((col >> 3) ^ (row & (C - 1))) << 4) + (col & 4) * 2) =
                pack4<T>(f(t, r), f(t, r + 1), f(t, r + 2), f(t, r + 3));
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32 * C / 64; ++i) {
        const int row = i * (64 / C) + l / C, c = l % C;
        const int64_t at = __shfl(offset, row);
        if (__shfl((int)in, row) && c * 8 < Dv)
            *reinterpret_cast<s16x8 *>(to + at + c * 8) = *reinterpret_cast<const s16x8 *>(own + row * (DV * 2) + ((c ^ (row & (C - 1))) << 4));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// 8 elements of a row at `p` as an operand, zeros where !in
__device__ __forceinline__ s16x8 load8(const void *p, bool in) {
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in) v = *reinterpret_cast<const s16x8 *>(p);
    return v;
}

template <typename T> __device__ __forceinline__ float lam_of(const Args &a, int head) {
    return a.lam_f32 ? ((const float *)a.lam)[head] : (float)((const T *)a.lam)[head];
}
__device__ __forceinline__ int64_t start_of(const Args &a, int b) { return a.q_start ? (int64_t)a.q_start[b] : a.Nk - a.Nq; }
__device__ __forceinline__ int64_t length_of(const Args &a, int b) {
    return a.kv_lengths ? min(a.Nk, max((int64_t)0, (int64_t)a.kv_lengths[b])) : a.Nk;
}

// ---------------------------------------------------------------------------------------------- forward
// NQ groups of 32 rows (queries), two waves each: one a map, so that a map's sums are all that a wave holds.  KT keys a tile, 32 of them
// at a time.  DT: head size rounded up to 32, 64, 128; values are up to 2 DT wide.  The running maximum is followed loosely: sums are
// scaled down only when it has grown by a factor of 2^8 (weights stay below 2^8 until then, and the final division takes care of them).
// Weights in two parts: both maps' common part goes out of the difference, what their weights were rounded by does not.  Rounded once, outputs
// of 4096 keys at lam = 0.5 were 1.55 times as far off as their own rounding leaves them, in f16 and in bf16, and the further the nearer the maps
// are to each other; in two parts they are as exact as that.  4 x 4096 queries and keys, 8 heads of 64, take 590 us with it, 395 without; 8 x 1 query over 16384
// keys 35 either way.
// Its products and exponentials take turns more than they overlap, and the chip's power bounds both: 590 us (1160 Tflop/s of products, the second parts'
// among them) with four waves a SIMD, for which heads of 64 make do with tiles of 32 keys and 128 registers; 640 with two.  (8192 causal tokens of one
// sequence, 8 heads: 347 and 372.)  Both maps in one wave took half as
// long again as one map a wave.
// Few queries are bound by their keys and values: 35 us for 178 MB (5.1 TB/s; a large copy moves 5.1) with 8 x 16384 of them.
template <typename T, int DT, int NQ, int KT>
__global__ __launch_bounds__(128 * NQ, DT == 32 || (DT == 64 && NQ == 4) ? 4 : 2) void attention_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 2 * NQ;
    constexpr int K_BYTES = KT * CK * 16, V_BYTES = KT * CV * 16, STAGE = 2 * K_BYTES + V_BYTES;
    static_assert(NQ * 32 * DV * 2 <= 2 * STAGE && NQ * 8192 <= 2 * STAGE, "results go through the same memory");
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), m = w & 1, qw = w >> 1;

    // ---- which rows: (batch, group of query heads, tile of rows, part of the keys)
    const int64_t rows = a.Nq * a.heads_per_row;
    const int tiles = (int)((rows + 32 * NQ - 1) / (32 * NQ));
    const int groups = a.H / a.heads_per_row;
    int unit, tile;
    place(blockIdx.x, a.B * groups, tiles * a.splits, unit, tile);
    const int split = tile % a.splits, group = unit % groups, b = unit / groups;
    tile /= a.splits;
    const int hk = group * a.heads_per_row / (a.H / a.Hk);
    // a lane's row: its query and head
    struct Row { int64_t i; int head; bool in; };
    auto row_of = [&](int lane) __attribute__((always_inline)) {
        const int64_t row = (int64_t)tile * 32 * NQ + qw * 32 + (lane & 31);
        const bool in = row < rows;
        const int sub = in ? (int)(row / a.Nq) : 0;
        return Row{in ? row - (int64_t)sub * a.Nq : 0, group * a.heads_per_row + sub, in};
    };

    const int64_t start = start_of(a, b);
    const int len = (int)length_of(a, b);
    auto upto = [&](int64_t i) { return a.causal ? (int)min((int64_t)len, max((int64_t)0, start + i + 1)) : len; };   // keys that query i sees
    const Row mine = row_of(l);
    const int sees = mine.in ? upto(mine.i) : 0;
    // (rows of one head are in order; several heads in one tile: from the first query's keys to the last one's)
    const bool packed = a.heads_per_row > 1;
    const int most = upto(packed ? a.Nq - 1 : min(a.Nq - 1, (int64_t)(tile + 1) * 32 * NQ - 1));
    const int fewest = upto(packed ? 0 : (int64_t)tile * 32 * NQ + qw * 32);    // that every row of the wave sees
    const int j_begin = (int)((int64_t)split * a.split_keys), j_end = (int)min((int64_t)most, j_begin + a.split_keys);

    const T *kp = (const T *)a.k + (int64_t)b * a.kb + (int64_t)(2 * hk) * a.kh;
    const T *vp = (const T *)a.v + (int64_t)b * a.vb + (int64_t)hk * a.vh;
    Stager<KT, CK, NW> stage_k;
    Stager<KT, CV, NW, true> stage_v;
    stage_k.begin(a.kn, a.D / 8, w, l);
    stage_v.begin(a.vn, a.Dv / 8, w, l);
    // the tile that is copied next; what lies past the last key that any of its rows sees is not read
    int j_next = j_begin;
    const T *k_next = kp + j_begin * a.kn, *v_next = vp + j_begin * a.vn;
    const int64_t k_step = KT * a.kn, v_step = KT * a.vn;
    auto fetch = [&](char *to) __attribute__((always_inline)) {
        stage_k.copy(to, k_next, most - j_next, w);
        stage_k.copy(to + K_BYTES, k_next + a.kh, most - j_next, w);
        stage_v.copy(to + 2 * K_BYTES, v_next, most - j_next, w);
        k_next += k_step;
        v_next += v_step;
        j_next += KT;
    };
    if (j_begin < j_end) fetch(smem);

    // ---- queries: right operands, in registers
    s16x8 qf[DT / 16];
    {
        const T *p = (const T *)a.q + (int64_t)b * a.qb + mine.i * a.qn + (int64_t)(2 * mine.head + m) * a.qh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            qf[s] = load8(p + c * 8, mine.in && c * 8 < a.D);
        }
    }
    RowReader<CK> keys;
    ColumnReader<CV, true> values;
    keys.begin(l);
    values.begin(l);
    keys.at += m * K_BYTES;

    f32x16 acc[DV / 32];
    clear(acc);
    float top = kLowest, total = 0.f;
    const float to_log2 = a.scale * kLog2e;

    // One tile; the next one is on its way to `ahead`.  (__restrict__: the compiler would have it arrive before the first read of `now`.)
    auto turn = [&](char *__restrict__ ahead, const char *__restrict__ now, int j) __attribute__((always_inline)) {
        tile_there<NW>();
        if (j + KT < j_end) fetch(ahead);
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            f32x16 s[1];
            clear(s);
#pragma unroll
            for (int d = 0; d < DT / 16; ++d) s[0] = mfma32<T>(keys.read(now, t, d), qf[d], s[0]);
            if (j + 32 * t + 32 > fewest) {
                const int n = sees - j - 32 * t - 4 * h32;  // (rows of the other half of the lanes are 4 further down)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (tile_row(r, 0) >= n) s[0][r] = -INFINITY;
            }
            float high = s[0][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) high = fmaxf(high, s[0][r]);
            high = both_halves_max(high) * to_log2;
            if (__any(high > top + 8.0f)) {
                const float up = fmaxf(top, high), shrink = __builtin_amdgcn_exp2f(top - up);
                top = up;
                total *= shrink;
#pragma unroll
                for (int v = 0; v < DV / 32; ++v)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[v][r] *= shrink;
            }
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], to_log2, -top));
                sum += s[0][r];
            }
            total += sum;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const s16x8 pf = as_operand<T>(s[0], x), rest = rest_of<T>(s[0], pf, x);
#pragma unroll
                for (int v = 0; v < DV / 32; ++v) {
                    const s16x8 column = values.read(now + 2 * K_BYTES, 32 * t + 16 * x, v);
                    acc[v] = mfma32<T>(column, pf, acc[v]);
                    acc[v] = mfma32<T>(column, rest, acc[v]);
                }
            }
        }
    };
    __builtin_amdgcn_s_waitcnt(0);                          // (what came before the loop is there, or its turns would wait for as much)
    for (int j = j_begin; j < j_end; j += 2 * KT) {
        turn(smem + STAGE, smem, j);
        if (j + KT < j_end) turn(smem, smem + STAGE, j + KT);
    }
    total = both_halves_sum(total);

    // (asked for anew, so that nothing of the lane and its row is kept through the loop)
    const int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), half = lane >> 5;
    const auto [i, head, row_in] = row_of(lane);
    if (a.part) {                                           // unfinished sums of this part
        if (!row_in) return;
        float *to = a.part + ((((int64_t)b * a.H + head) * a.Nq + i) * a.splits + split) * (2 * a.Dv + 4);
#pragma unroll
        for (int t = 0; t < DV / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * t + tile_row(r, half);
                const f32x4 v = {acc[t][r], acc[t][r + 1], acc[t][r + 2], acc[t][r + 3]};
                if (d < a.Dv) *reinterpret_cast<f32x4 *>(to + m * a.Dv + d) = v;
            }
        if (half == 0) to[2 * a.Dv + m] = top, to[2 * a.Dv + 2 + m] = total;
        return;
    }
    const float weight = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
    for (int t = 0; t < DV / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] *= weight;
    const int64_t at = (((int64_t)b * a.Nq + i) * a.H + head) * a.Dv;
    const float lam = lam_of<T>(a, head);
    // the first map's wave takes off the second's, two tiles at a time
#pragma unroll
    for (int t = 0; t < DV / 32; t += 2) {
        tile_there<NW>();                                   // (every wave is through with what lies there)
        f32x4 *by = reinterpret_cast<f32x4 *>(smem) + qw * 512 + lane;
        if (m)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const f32x16 &x = acc[t + r / 4];
                const int e = r % 4 * 4;
                by[r * 64] = (f32x4){x[e], x[e + 1], x[e + 2], x[e + 3]};
            }
        tile_there<NW>();
        if (!m)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const f32x4 y = by[r * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t + r / 4][r % 4 * 4 + e] -= lam * y[e];
            }
    }
    char *own = smem + qw * 32 * DV * 2;
    tile_there<NW>();
    if (!m) store_rows<T, DV>(own, (T *)a.o, at, row_in, a.Dv, lane, [&](int t, int r) { return acc[t][r]; });
    if (a.o2) {
        tile_there<NW>();
        if (m) store_rows<T, DV>(own, (T *)a.o2, at, row_in, a.Dv, lane, [&](int t, int r) { return acc[t][r]; });
    }
    if (a.lse && row_in && half == 0)
        a.lse[((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i] = total == 0.f ? INFINITY : top + __log2f(total);
}

// Joins the parts of a row: a workgroup a row, a thread a value of one map.  The parts' weights first, in LDS.
constexpr int MAX_SPLITS = 128;
template <typename T> __global__ __launch_bounds__(512) void attention_join_kernel(Args a) {
    __shared__ float weight[2][MAX_SPLITS], first[256];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, width = 2 * a.Dv + 4;
    const float *p = a.part + row * a.splits * width;
    if (tid < 128) {                                        // one wave a map
        const int m = tid >> 6, l = tid & 63;
        float t[2], s[2], top = kLowest, total = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool in = l + 64 * u < a.splits;
            t[u] = in ? p[(int64_t)(l + 64 * u) * width + 2 * a.Dv + m] : kLowest;
            s[u] = in ? p[(int64_t)(l + 64 * u) * width + 2 * a.Dv + 2 + m] : 0.f;
            top = fmaxf(top, t[u]);
        }
#pragma unroll
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            t[u] = __builtin_amdgcn_exp2f(t[u] - top);
            total += s[u] * t[u];
        }
#pragma unroll
        for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
#pragma unroll
        for (int u = 0; u < 2; ++u) weight[m][l + 64 * u] = total == 0.f ? 0.f : t[u] / total;
        if (a.lse && l == 0) {
            const int64_t i = row % a.Nq, bh = row / a.Nq;
            a.lse[(2 * bh + m) * a.Nq + i] = total == 0.f ? INFINITY : top + __log2f(total);
        }
    }
    __syncthreads();
    const int m = tid >> 8, d = tid & 255;
    float x = 0.f;
    if (d < a.Dv) {
#pragma unroll 8
        for (int s = 0; s < a.splits; ++s) x += p[(int64_t)s * width + m * a.Dv + d] * weight[m][s];
    }
    if (m == 1) first[d] = x;
    __syncthreads();
    if (m == 0 && d < a.Dv) {
        const int64_t i = row % a.Nq, bh = row / a.Nq;
        const int head = (int)(bh % a.H);
        const int64_t at = ((bh / a.H * a.Nq + i) * a.H + head) * a.Dv + d;
        ((T *)a.o)[at] = (T)(x - lam_of<T>(a, head) * first[d]);
        if (a.o2) ((T *)a.o2)[at] = (T)first[d];
    }
}

// ---------------------------------------------------------------------------------------------- centres of the gradients
// D1 and D2, which both kernels of gradients need first.  dP - D cancels in rows whose weight is nearly all on a few keys, and then what D
// is off by is what dq shows: from outputs rounded to 16 bits, D' = do . o_m, scores of deviation 6 gave a bf16 dq as far off as it is long.
// So a pass over the keys forms  D_m = D' + sum_j P_mj (dP_j - D')  in 32 bits.  (Of the differences: what log-sum-exp of large scores is
// off by makes the weights' sum 1 + e, and counts here as e (D - D'), not as e D.)
// 72 us for 4 x 2047 causal tokens and 8 heads of 64 over 128 of ragged lengths (21 Gflop, 290 Tflop/s): exponentials, the arithmetic around
// them and the products take about as long as one another, and three waves a SIMD run them beside one another.  Done in the next kernel, with the registers that its
// sums hold, it took as long with two.
template <typename T, int DT, int KT>
__global__ __launch_bounds__(THREADS, DT == 32 ? 4 : DT == 64 ? 3 : 2) void attention_delta_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 4;
    constexpr int K_BYTES = KT * CK * 16, V_BYTES = KT * CV * 16, STAGE = 2 * K_BYTES + V_BYTES;
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)((a.Nq + 127) / 128);
    int unit, tile;
    place(blockIdx.x, a.B * a.H, tiles, unit, tile);
    const int head = unit % a.H, b = unit / a.H;
    const int hk = head / (a.H / a.Hk);
    const int64_t row = (int64_t)tile * 128 + w * 32 + (l & 31);
    const bool row_in = row < a.Nq;
    const int64_t i = row_in ? row : 0;
    const int64_t start = start_of(a, b);
    const int len = (int)length_of(a, b);
    auto upto = [&](int64_t i) { return a.causal ? (int)min((int64_t)len, max((int64_t)0, start + i + 1)) : len; };
    const int sees = row_in ? upto(i) : 0, j_end = upto(min(a.Nq - 1, (int64_t)tile * 128 + 127)), fewest = upto((int64_t)tile * 128 + w * 32);
    s16x8 qf[2][DT / 16], gf[DV / 16];
    const float lam = lam_of<T>(a, head);
    float delta[2] = {0.f, 0.f};
    {
        const T *g = (const T *)a.dout + (int64_t)b * a.dob + i * a.don + (int64_t)head * a.doh;
        const int64_t at = (((int64_t)b * a.Nq + i) * a.H + head) * a.Dv;
#pragma unroll
        for (int s = 0; s < DV / 16; ++s) {
            const int c = 2 * s + h32;
            const bool in = row_in && c * 8 < a.Dv;
            gf[s] = load8(g + c * 8, in);
            const s16x8 o = load8((const T *)a.o + at + c * 8, in), o2 = load8((const T *)a.o2 + at + c * 8, in);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const short gs = gf[s][e], os = o[e], ps = o2[e];
                const float ge = widen<T>(gs);
                delta[0] += ge * widen<T>(os);
                delta[1] += ge * widen<T>(ps);
            }
        }
        delta[0] = both_halves_sum(delta[0]);
        delta[1] = both_halves_sum(delta[1]);
        delta[0] += lam * delta[1];                         // (o + lam o2 is the first map's output)
    }
    __builtin_amdgcn_sched_barrier(0);                      // (queries beside the outputs have no registers in heads of 128)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const T *p = (const T *)a.q + (int64_t)b * a.qb + i * a.qn + (int64_t)(2 * head + m) * a.qh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            qf[m][s] = load8(p + c * 8, row_in && c * 8 < a.D);
        }
    }
    float lse[2], off[2] = {0.f, 0.f}, peak = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) lse[m] = row_in ? a.lse[((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i] : INFINITY;

    const float to_log2 = a.scale * kLog2e;
    const T *kp = (const T *)a.k + (int64_t)b * a.kb + (int64_t)(2 * hk) * a.kh;
    const T *vp = (const T *)a.v + (int64_t)b * a.vb + (int64_t)hk * a.vh;
    Stager<KT, CK, NW> stage_k;
    Stager<KT, CV, NW> stage_v;
    stage_k.begin(a.kn, a.D / 8, w, l);
    stage_v.begin(a.vn, a.Dv / 8, w, l);
    auto fetch = [&](char *to, int j) __attribute__((always_inline)) {
        stage_k.copy(to, kp + j * a.kn, j_end - j, w);
        stage_k.copy(to + K_BYTES, kp + a.kh + j * a.kn, j_end - j, w);
        stage_v.copy(to + 2 * K_BYTES, vp + j * a.vn, j_end - j, w);
    };
    RowReader<CK> keys;
    RowReader<CV> values;
    keys.begin(l);
    values.begin(l);
    if (0 < j_end) fetch(smem, 0);
    auto turn = [&](char *__restrict__ ahead, const char *__restrict__ now, int j) __attribute__((always_inline)) {
        tile_there<NW>();
        if (j + KT < j_end) fetch(ahead, j + KT);
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            f32x16 dp[1];
            clear(dp);
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) dp[0] = mfma32<T>(values.read(now + 2 * K_BYTES, t, d), gf[d], dp[0]);
#pragma unroll
            for (int r = 0; r < 16; r += 2) peak = fmaxf(peak, fmaxf(fabsf(dp[0][r]), fabsf(dp[0][r + 1])));
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                f32x16 s[1];
                clear(s);
#pragma unroll
                for (int d = 0; d < DT / 16; ++d) s[0] = mfma32<T>(keys.read(now + m * K_BYTES, t, d), qf[m][d], s[0]);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], to_log2, -lse[m]));
                if (j + 32 * t + 32 > fewest) {
                    const int n = sees - j - 32 * t - 4 * h32;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (tile_row(r, 0) >= n) s[0][r] = 0.f;
                }
                float sum[2] = {0.f, 0.f};                  // (two chains: a sum waits for the one before)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[r & 1] = __builtin_fmaf(s[0][r], dp[0][r] - delta[m], sum[r & 1]);
                off[m] += sum[0] + sum[1];
            }
        }
    };
    __builtin_amdgcn_s_waitcnt(0);                          // (what came before the loop is there, or its turns would wait for as much)
    for (int j = 0; j < j_end; j += 2 * KT) {
        turn(smem + STAGE, smem, j);
        if (j + KT < j_end) turn(smem, smem + STAGE, j + KT);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        delta[m] += both_halves_sum(off[m]);
        if (row_in && h32 == 0) a.delta[((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i] = delta[m];
    }
    float sum = delta[1];                                   // (0 for rows past the end)
#pragma unroll
    for (int x = 1; x < 32; x *= 2) sum += __shfl_xor(sum, x);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) peak = fmaxf(peak, __shfl_xor(peak, x));
    if (l == 0) {
        a.d2_sums[(((int64_t)head * a.B + b) * tiles + tile) * NW + w] = sum;
        a.peaks[(((int64_t)b * a.H + head) * tiles + tile) * NW + w] = peak * fmaxf(1.0f, fabsf(lam));
    }
}

// ---------------------------------------------------------------------------------------------- gradients of the queries
// As the forward pass: a lane holds one query, dS^T is at once the right operand of  dq^T += k^T dS^T.
// dS in two parts: rounded once, dq of bf16 keys that have six times their deviation in common was off by 1.2e-2 of its length (storing it: 1.6e-3).  88 us for 4 x 2047
// causal tokens and 8 heads of 64 over 128 of ragged lengths (42 Gflop, 470 Tflop/s), 73 with dS in one part: half of a wave's time goes to exponentials and the
// arithmetic between the products.
template <typename T, int DT, int KT>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(DT == 128 ? 1 : 2, DT == 128 ? 1 : 2))) void attention_dq_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 4;
    constexpr int K_BYTES = KT * CK * 16, V_BYTES = KT * CV * 16, STAGE = 2 * K_BYTES + V_BYTES;
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    static_assert(NW * 32 * DT * 2 <= 2 * STAGE, "results go through the same memory");
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)((a.Nq + 127) / 128);
    int unit, tile;
    place(blockIdx.x, a.B * a.H, tiles, unit, tile);
    const int head = unit % a.H, b = unit / a.H;
    const int hk = head / (a.H / a.Hk);
    const int64_t row = (int64_t)tile * 128 + w * 32 + (l & 31);
    const bool row_in = row < a.Nq;
    const int64_t i = row_in ? row : 0;
    const int64_t start = start_of(a, b);
    const int len = (int)length_of(a, b);
    auto upto = [&](int64_t i) { return a.causal ? (int)min((int64_t)len, max((int64_t)0, start + i + 1)) : len; };
    const int sees = row_in ? upto(i) : 0, j_end = upto(min(a.Nq - 1, (int64_t)tile * 128 + 127)), fewest = upto((int64_t)tile * 128 + w * 32);
    const bool single = __any(sees == 1);
    s16x8 qf[2][DT / 16], gf[DV / 16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const T *p = (const T *)a.q + (int64_t)b * a.qb + i * a.qn + (int64_t)(2 * head + m) * a.qh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            qf[m][s] = load8(p + c * 8, row_in && c * 8 < a.D);
        }
    }
    const float lam = lam_of<T>(a, head), step = a.steps[b * a.Hk + hk];
    {
        const T *g = (const T *)a.dout + (int64_t)b * a.dob + i * a.don + (int64_t)head * a.doh;
#pragma unroll
        for (int s = 0; s < DV / 16; ++s) {
            const int c = 2 * s + h32;
            gf[s] = load8(g + c * 8, row_in && c * 8 < a.Dv);
        }
    }
    float lse[2], delta[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int64_t at = ((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i;
        lse[m] = row_in ? a.lse[at] : INFINITY;
        delta[m] = row_in ? step * a.delta[at] : 0.f;
    }

    f32x16 acc[2][DT / 32];
    clear(acc[0]);
    clear(acc[1]);
    const float to_log2 = a.scale * kLog2e;
    const T *kp = (const T *)a.k + (int64_t)b * a.kb + (int64_t)(2 * hk) * a.kh;
    const T *vp = (const T *)a.v + (int64_t)b * a.vb + (int64_t)hk * a.vh;
    Stager<KT, CK, NW> stage_k;
    Stager<KT, CV, NW> stage_v;
    stage_k.begin(a.kn, a.D / 8, w, l);
    stage_v.begin(a.vn, a.Dv / 8, w, l);
    auto fetch = [&](char *to, int j) __attribute__((always_inline)) {
        stage_k.copy(to, kp + j * a.kn, j_end - j, w);
        stage_k.copy(to + K_BYTES, kp + a.kh + j * a.kn, j_end - j, w);
        stage_v.copy(to + 2 * K_BYTES, vp + j * a.vn, j_end - j, w);
    };
    RowReader<CK> keys;
    RowReader<CV> values;
    ColumnReader<CK> key_columns;
    keys.begin(l);
    values.begin(l);
    key_columns.begin(l);
    if (0 < j_end) fetch(smem, 0);
    auto turn = [&](char *__restrict__ ahead, const char *__restrict__ now, int j) __attribute__((always_inline)) {
        tile_there<NW>();
        if (j + KT < j_end) fetch(ahead, j + KT);
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            const bool masked = j + 32 * t + 32 > fewest || single;
            f32x16 dp[1];
            clear(dp);
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) dp[0] = mfma32<T>(values.read(now + 2 * K_BYTES, t, d), gf[d], dp[0]);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                f32x16 s[1];
                clear(s);
#pragma unroll
                for (int d = 0; d < DT / 16; ++d) s[0] = mfma32<T>(keys.read(now + m * K_BYTES, t, d), qf[m][d], s[0]);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], to_log2, -lse[m])) * __builtin_fmaf(dp[0][r], step, -delta[m]);
                if (masked) {                               // (a row that sees one key has weight 1 there whatever its score)
                    const int n = sees == 1 ? 0 : sees - j - 32 * t - 4 * h32;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (tile_row(r, 0) >= n) s[0][r] = 0.f;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const s16x8 ds = as_operand<T>(s[0], x), rest = rest_of<T>(s[0], ds, x);
#pragma unroll
                    for (int d = 0; d < DT / 32; ++d) {
                        const s16x8 column = key_columns.read(now + m * K_BYTES, 32 * t + 16 * x, d);
                        acc[m][d] = mfma32<T>(column, ds, acc[m][d]);
                        acc[m][d] = mfma32<T>(column, rest, acc[m][d]);
                    }
                }
            }
        }
    };
    __builtin_amdgcn_s_waitcnt(0);                          // (what came before the loop is there, or its turns would wait for as much)
    for (int j = 0; j < j_end; j += 2 * KT) {
        turn(smem + STAGE, smem, j);
        if (j + KT < j_end) turn(smem, smem + STAGE, j + KT);
    }
    tile_there<NW>();
    char *own = smem + w * 32 * DT * 2;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float f = (m ? -lam * a.scale : a.scale) / step;
        store_rows<T, DT>(own, (T *)a.dq, (((int64_t)b * a.Nq + i) * 2 * a.H + 2 * head + m) * a.D, row_in, a.D, l,
                          [&](int t, int r) { return acc[m][t][r] * f; });
    }
}

// ---------------------------------------------------------------------------------------------- gradients of keys and values
// The other way round: a lane holds one key, scores have queries down and keys across, W = P1 - lam P2 and dS_m are the right operands
// of  dv^T += do^T W  and  dk_m^T += q_m^T dS_m.  A workgroup owns 64 keys, whose operands stay in registers while the queries of every
// head that reads them pass through LDS, 64 at a time, so shared heads' gradients are summed here.  Two waves take the first half of the
// queries in a tile, two the second; their sums are added at the end, in order.
// WHAT: 1 dv, 2 dk, 3 both.  Of heads of 128 dk alone takes a wave's 512 registers: there dv and dk are summed by a launch each.
// 127 us for 4 x 2047 causal tokens, 8 heads of 64 over 128 and 4 key heads, ragged (41 Gflop, 330 Tflop/s), bound like the kernel above; one wave
// a SIMD, because dk, dv and the operands of 32 keys take 410 registers.
template <typename T, int DT, int WHAT>
__global__ __launch_bounds__(THREADS, 1) void attention_dkv_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 4, QT = 64;
    constexpr bool VALUES = WHAT & 1, KEYS = (WHAT & 2) != 0;
    constexpr int Q_BYTES = QT * CK * 16, G_BYTES = QT * CV * 16, STATS = 4 * QT * 4, STAGE = 2 * Q_BYTES + G_BYTES + STATS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), kw = w & 1, qw = w >> 1;
    const int tiles = (int)((a.Nk + 63) / 64);
    // (with a causal mask the first keys are seen by the most queries: they begin first)
    int id = blockIdx.x;
    const int hk = id % a.Hk; id /= a.Hk;
    const int b = id % a.B, tile = id / a.B;
    if (tile >= tiles) return;
    const int per = a.H / a.Hk;
    // (no key or query has a number above 2^29)
    const int start = (int)max(-((int64_t)1 << 29), min((int64_t)1 << 29, start_of(a, b))), nq = (int)a.Nq;
    // keys that some query sees
    const int length = (int)length_of(a, b), len = a.causal ? max(0, min(length, start + nq)) : length, first_key = tile * 64, key0 = first_key + kw * 32, key = key0 + (l & 31);
    const bool key_in = key < len;

    // queries that see any key of this workgroup: from i_first on
    int i_first = 0;
    if (a.causal) i_first = max(0, first_key - start) / QT * QT;
    if (first_key >= len) i_first = nq;
    const int per_head = i_first < nq ? (nq - i_first + QT - 1) / QT : 0;
    int steps = per_head * per;

    // the tile of queries that is copied next, and the ways to the next tile and, from behind the last one, to the next head's first
    Stager<QT, CK, NW> stage_q;
    Stager<QT, CV, NW> stage_g;
    stage_q.begin(a.qn, a.D / 8, w, l);
    stage_g.begin(a.don, a.Dv / 8, w, l);
    int i_next = i_first;
    const T *q_next = (const T *)a.q + (int64_t)b * a.qb + i_first * a.qn + (int64_t)(2 * hk * per) * a.qh;
    const T *d_next = (const T *)a.dout + (int64_t)b * a.dob + i_first * a.don + (int64_t)(hk * per) * a.doh;
    // one of lse1, lse2, D1, D2 a wave.  (Queries past the end have zeros everywhere: their weight of 1 meets do = 0.)
    const float *s_next = (w < 2 ? a.lse : a.delta) + ((int64_t)b * 2 * a.H + 2 * (hk * per) + (w & 1)) * a.Nq + i_first;
    const int64_t q_step = QT * a.qn, d_step = QT * a.don;
    const int64_t q_turn = 2 * a.qh - per_head * q_step, d_turn = a.doh - per_head * d_step, s_turn = 2 * a.Nq - per_head * QT;
    auto fetch = [&](char *to) __attribute__((always_inline)) {
        const int in = min(QT, nq - i_next);
        stage_q.copy(to, q_next, in, w);
        stage_q.copy(to + Q_BYTES, q_next + a.qh, in, w);
        stage_g.copy(to + 2 * Q_BYTES, d_next, in, w);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(uniform_rsrc(s_next, kAnywhere), (lds_ptr_t)(to + 2 * Q_BYTES + G_BYTES + w * QT * 4), 4,
                                                 l < in ? (uint32_t)l * 4u : kNowhere, 0, 0, 0);
        q_next += q_step;
        d_next += d_step;
        s_next += QT;
        i_next += QT;
        if (i_next >= nq) {
            q_next += q_turn;
            d_next += d_turn;
            s_next += s_turn;
            i_next = i_first;
        }
    };
    if (steps) fetch(smem);

    s16x8 kf[2][DT / 16], vf[KEYS ? DV / 16 : 1];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const T *p = (const T *)a.k + (int64_t)b * a.kb + (int64_t)(key_in ? key : 0) * a.kn + (int64_t)(2 * hk + m) * a.kh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            kf[m][s] = load8(p + c * 8, key_in && c * 8 < a.D);
        }
    }
    if constexpr (KEYS) {
        const T *p = (const T *)a.v + (int64_t)b * a.vb + (int64_t)(key_in ? key : 0) * a.vn + (int64_t)hk * a.vh;
#pragma unroll
        for (int s = 0; s < DV / 16; ++s) {
            const int c = 2 * s + h32;
            vf[s] = load8(p + c * 8, key_in && c * 8 < a.Dv);
        }
    }
    RowReader<CK> queries;
    RowReader<CV> grads;
    ColumnReader<CK> query_columns;
    ColumnReader<CV> grad_columns;
    queries.begin(l);
    grads.begin(l);
    query_columns.begin(l);
    grad_columns.begin(l);
    f32x16 dk[KEYS ? 2 : 1][DT / 32], dv[VALUES ? DV / 32 : 1];
    clear(dk[0]);
    clear(dk[KEYS ? 1 : 0]);
    clear(dv);
    const float to_log2 = a.scale * kLog2e;

    int g = 0;
    int i0 = i_first;
    // (made uniform, and thereby waited for, where it is read: a wait for it later on would be one for the copies as well)
    auto lam_of_head = [&](int head) {
        const float x = lam_of<T>(a, head);
        return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
    };
    float lam = lam_of_head(hk * per);
    const float step = a.steps[b * a.Hk + hk];
    auto turn = [&](char *__restrict__ ahead, const char *__restrict__ now) __attribute__((always_inline)) {
        tile_there<NW>();
        if (steps > 1) fetch(ahead);
        const char *gs = now + 2 * Q_BYTES;
        const float *stats = reinterpret_cast<const float *>(gs + G_BYTES) + 32 * qw + 4 * h32;
        // the last key that the first of these queries sees (clamped: only its place among the keys counts)
        const int last0 = a.causal ? max(-64, start + i0 + 32 * qw) : 1 << 30;
        const int last = last0 + 4 * h32;
        // some pair is hidden, or some row sees one key only
        const bool masked = key0 + 32 > len || key0 + 31 > last0 || len == 1 || last0 <= 0;
        // One wave a SIMD has nothing else to do while it waits: reads go out in groups, ahead of what needs them.
        s16x8 rows[2][DT / 16], grad_rows[KEYS ? DV / 16 : 1];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < DT / 16; ++d) rows[m][d] = queries.read(now + m * Q_BYTES, qw, d);
        if constexpr (KEYS)
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) grad_rows[d] = grads.read(gs, qw, d);
        f32x4 ls[2][4], de[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ls[m][r] = *reinterpret_cast<const f32x4 *>(stats + m * QT + 8 * r);
                if constexpr (KEYS) de[m][r] = *reinterpret_cast<const f32x4 *>(stats + (2 + m) * QT + 8 * r);
            }
        if constexpr (DT <= 64) __builtin_amdgcn_sched_barrier(0);
        f32x16 dp[1], s[2];
        clear(dp);
        clear(s);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < DT / 16; ++d) s[m] = mfma32<T>(rows[m][d], kf[m][d], s[m]);
        if constexpr (KEYS)
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) dp[0] = mfma32<T>(grad_rows[d], vf[d], dp[0]);
        s16x8 query_cols[KEYS ? 2 : 1][2][DT / 32], grad_cols[VALUES ? 2 : 1][DV / 32];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if constexpr (KEYS)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int d = 0; d < DT / 32; ++d) query_cols[m][x][d] = query_columns.read(now + m * Q_BYTES, 32 * qw + 16 * x, d);
            if constexpr (VALUES)
#pragma unroll
                for (int d = 0; d < DV / 32; ++d) grad_cols[x][d] = grad_columns.read(gs, 32 * qw + 16 * x, d);
        }
        if constexpr (DT <= 64) __builtin_amdgcn_sched_barrier(0);
        f32x16 p[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[m][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][r], to_log2, -ls[m][r / 4][r % 4]));
                if constexpr (KEYS) s[m][r] = p[m][r] * (dp[0][r] - de[m][r / 4][r % 4]);
            }
        if (masked) {
            const int beyond = key < len ? key - last : 1 << 30;
#pragma unroll
            for (int r = 0; r < 16; ++r) {                  // query tile_row(r, 0) of the half sees keys up to last + that
                const bool hidden = beyond > tile_row(r, 0), none = hidden | (-last == tile_row(r, 0)) | (len == 1);
#pragma unroll
                for (int m = 0; m < 2; ++m) {               // (selections: as branches they are 3000 instructions)
                    p[m][r] = hidden ? 0.f : p[m][r];
                    s[m][r] = none ? 0.f : s[m][r];
                }
            }
        }
        if constexpr (KEYS)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!x)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[m][r] *= m ? -lam * step : step;
                    const s16x8 ds = as_operand<T>(s[m], x);
#pragma unroll
                    for (int d = 0; d < DT / 32; ++d) dk[m][d] = mfma32<T>(query_cols[m][x][d], ds, dk[m][d]);
                }
        if constexpr (VALUES) {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[0][r] -= lam * p[1][r];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const s16x8 wf = as_operand<T>(p[0], x);
#pragma unroll
                for (int d = 0; d < DV / 32; ++d) dv[d] = mfma32<T>(grad_cols[x][d], wf, dv[d]);
            }
        }
        i0 += QT;
        if (--steps && i0 >= nq) {
            i0 = i_first;
            lam = lam_of_head(hk * per + ++g);
        }
    };
    __builtin_amdgcn_s_waitcnt(0);                          // (what came before the loop is there, or its turns would wait for as much)
    while (steps > 0) {
        turn(smem + STAGE, smem);
        if (steps > 0) turn(smem, smem + STAGE);
    }
    // ---- the second half's sums are added to the first's, 32 registers of a lane at a time
    auto add = [&](f32x16 &x, f32x16 &y) __attribute__((always_inline)) {
        tile_there<NW>();
        f32x4 *at = reinterpret_cast<f32x4 *>(smem) + kw * 512 + l;
        if (qw) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                at[r * 64] = (f32x4){x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
                at[(4 + r) * 64] = (f32x4){y[4 * r], y[4 * r + 1], y[4 * r + 2], y[4 * r + 3]};
            }
        }
        tile_there<NW>();
        if (!qw) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 u = at[r * 64], v = at[(4 + r) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * r + e] += u[e], y[4 * r + e] += v[e];
            }
        }
    };
    if constexpr (VALUES)
#pragma unroll
        for (int d = 0; d < DV / 32; d += 2) add(dv[d], dv[d + 1]);
    if constexpr (KEYS)
#pragma unroll
        for (int d = 0; d < DT / 32; ++d) add(dk[0][d], dk[1][d]);
    tile_there<NW>();
    if (qw) return;
    const float back = a.scale / step;
    char *own = smem + kw * 32 * DV * 2;
    const bool to_write = key < a.Nk;
    const int64_t at = (int64_t)b * a.Nk + (to_write ? key : 0);
    if constexpr (KEYS)
#pragma unroll
        for (int m = 0; m < 2; ++m)
            store_rows<T, DT>(own, (T *)a.dk, (at * 2 * a.Hk + 2 * hk + m) * a.D, to_write, a.D, l, [&](int t, int r) { return dk[m][t][r] * back; });
    if constexpr (VALUES) store_rows<T, DV>(own, (T *)a.dv, (at * a.Hk + hk) * a.Dv, to_write, a.Dv, l, [&](int t, int r) { return dv[t][r]; });
}

// What the kernel of the centres has left of each 32 queries, joined in a fixed order; a workgroup each.
// dlam[h] = - sum over sequences and queries of D2.  4.5 us for 8 heads of 8188 queries, where reading all of D2 here took 11.
// Behind them, for each sequence and key head: a power of two by which |dP - D| max(1, |lam|), at most twice the largest |dP|, stays within 2^15 in all its
// queries.  dS goes to the matrix units multiplied by it: f16, which ends at 65504 and has all its digits down to 2^-14, then neither overflows nor loses
// digits of weights above 2^-29, whatever factor the loss is scaled by.  (bf16 has the same exponents as 32 bits: to it this changes nothing.)
template <typename T> __global__ __launch_bounds__(THREADS) void attention_totals_kernel(Args a) {
    __shared__ float part[THREADS];
    const bool sums = blockIdx.x < a.H;
    const int64_t runs = (a.Nq + 127) / 128 * 4, n = runs * (sums ? a.B : a.H / a.Hk);
    const float *of = sums ? a.d2_sums + blockIdx.x * n : a.peaks + (blockIdx.x - a.H) * n;
    float x = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += THREADS) x = sums ? x + of[i] : fmaxf(x, of[i]);
    part[threadIdx.x] = x;
    __syncthreads();
    for (int y = THREADS / 2; y > 0; y /= 2) {
        if (threadIdx.x < y) {
            const float u = part[threadIdx.x], v = part[threadIdx.x + y];
            part[threadIdx.x] = sums ? u + v : fmaxf(u, v);
        }
        __syncthreads();
    }
    if (threadIdx.x) return;
    x = part[0];
    if (!sums) {
        int e = 0;                                          // x < 2^e
        if (x > 0.f && x <= 3.4e38f) frexpf(x, &e);
        a.steps[blockIdx.x - a.H] = ldexpf(1.0f, min(100, max(-100, 14 - e)));
    } else if (a.lam_f32) ((float *)a.dlam)[blockIdx.x] = -x;
    else ((T *)a.dlam)[blockIdx.x] = (T)-x;
}

// ---------------------------------------------------------------------------------------------- host side
struct Plan {
    int heads_per_row, waves, splits;
    int64_t split_keys, blocks;
};

int padded(int D, int Dv) { const int d = D > (Dv + 1) / 2 ? D : (Dv + 1) / 2; return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

Plan plan_of(const bndm_attention_shape &s) {
    Plan p;
    // few queries: all heads that share a key head in one tile of rows, so that their keys are read once
    const int per = s.H / s.Hk;
    p.heads_per_row = s.Nq * per <= 32 ? per : 1;
    const int64_t rows = s.Nq * p.heads_per_row;
    p.waves = rows <= 32 ? 1 : 4;
    const int64_t tiles = ceil_div64(rows, 32 * p.waves) * (s.H / p.heads_per_row) * s.B;
    // parts of the keys: as many as give 256 CUs four workgroups of two waves or one of eight, of 256 keys at least
    const int64_t want = p.waves == 1 ? 1024 : 256;
    int64_t splits = tiles >= want ? 1 : ceil_div64(want, tiles);
    const int64_t most = s.Nk / 256 < 1 ? 1 : s.Nk / 256;
    if (splits > most) splits = most;
    if (splits > MAX_SPLITS) splits = MAX_SPLITS;
    p.split_keys = ceil_div64(ceil_div64(s.Nk, splits), 64) * 64;
    if (p.split_keys < 64) p.split_keys = 64;
    p.splits = (int)ceil_div64(s.Nk > 0 ? s.Nk : 1, p.split_keys);
    p.blocks = tiles * p.splits;
    return p;
}

template <typename F> int allow_lds(F kernel, int bytes, const char *what) {
    if (bytes <= 65536) return 0;
    const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) return 0;
    (void)hipGetLastError();
    tokens_error("%s: %d bytes of LDS: %s", what, bytes, hipGetErrorString(e));
    return (int)e;
}

template <typename T, int DT> int forward(const Args &a, const Plan &p, hipStream_t stream) {
    constexpr int KT = DT == 32 ? 64 : 32;
    if (p.waves == 1) hipLaunchKernelGGL((attention_kernel<T, DT, 1, 32>), dim3((unsigned)p.blocks), dim3(128), 0, stream, a);
    else hipLaunchKernelGGL((attention_kernel<T, DT, 4, KT>), dim3((unsigned)p.blocks), dim3(512), 0, stream, a);
    if (int rc = tokens_launch_status("attention")) return rc;
    if (a.part) {
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)((int64_t)a.B * a.H * a.Nq)), dim3(512), 0, stream, a);
        return tokens_launch_status("attention join");
    }
    return 0;
}

template <typename T, int DT, int WHAT> int launch_dkv(const Args &a, hipStream_t stream) {
    constexpr int LDS = 2 * (64 * DT * 8 + 4 * 64 * 4);
    if (int rc = allow_lds(attention_dkv_kernel<T, DT, WHAT>, LDS, "attention dkv")) return rc;
    hipLaunchKernelGGL((attention_dkv_kernel<T, DT, WHAT>), dim3((unsigned)(ceil_div64(a.Nk, 64) * a.Hk * a.B)), dim3(THREADS), LDS, stream, a);
    return tokens_launch_status("attention dkv");
}

template <typename T, int DT> int backward(const Args &a, hipStream_t stream) {
    constexpr int KT = DT == 128 ? 32 : 64;
    const int64_t nq = ceil_div64(a.Nq, 128) * a.H * a.B;
    hipLaunchKernelGGL((attention_delta_kernel<T, DT, 32>), dim3((unsigned)nq), dim3(THREADS), 0, stream, a);
    if (int rc = tokens_launch_status("attention delta")) return rc;
    hipLaunchKernelGGL((attention_totals_kernel<T>), dim3((unsigned)(a.H + a.B * a.Hk)), dim3(THREADS), 0, stream, a);
    if (int rc = tokens_launch_status("attention totals")) return rc;
    hipLaunchKernelGGL((attention_dq_kernel<T, DT, KT>), dim3((unsigned)nq), dim3(THREADS), 0, stream, a);
    if (int rc = tokens_launch_status("attention dq")) return rc;
    if (a.Nk == 0) return 0;
    if constexpr (DT == 128) {
        if (int rc = launch_dkv<T, DT, 1>(a, stream)) return rc;
        return launch_dkv<T, DT, 2>(a, stream);
    } else return launch_dkv<T, DT, 3>(a, stream);
}

int check(const char *what, const bndm_attention_shape *s) {
    TOKENS_REQUIRE(s, "%s: NULL shape", what);
    TOKENS_REQUIRE(s->B >= 0 && s->Nq >= 0 && s->Nk >= 0 && s->B <= (1 << 20) && s->Nq <= (1 << 29) && s->Nk <= (1 << 29), "%s: sizes", what);
    TOKENS_REQUIRE(s->H >= 1 && s->Hk >= 1 && s->H % s->Hk == 0 && s->H <= 4096, "%s: %d heads over %d key heads", what, s->H, s->Hk);
    TOKENS_REQUIRE(s->D >= 8 && s->D <= 128 && s->D % 8 == 0, "%s: head size %d: a multiple of 8 up to 128", what, s->D);
    TOKENS_REQUIRE(s->Dv >= 8 && s->Dv <= 256 && s->Dv % 8 == 0, "%s: value size %d: a multiple of 8 up to 256", what, s->Dv);
    TOKENS_REQUIRE(s->dtype == BNDM_DTYPE_F16 || s->dtype == BNDM_DTYPE_BF16, "%s: dtype %d (f16 and bf16 only)", what, s->dtype);
    TOKENS_REQUIRE(std::isfinite(s->scale) && s->scale > 0.f, "%s: scale must be a positive number", what);
    const int64_t *all[3] = {s->q_strides, s->k_strides, s->v_strides};
    for (int t = 0; t < 3; ++t)
        for (int i = 0; i < 3; ++i)
            TOKENS_REQUIRE(all[t][i] >= 0 && all[t][i] % 8 == 0 && (i != 1 || all[t][i] <= (1 << 23)), "%s: stride %lld: a multiple of 8, between tokens up to 2^23",
                           what, (long long)all[t][i]);
    TOKENS_REQUIRE(ceil_div64(s->Nq, 32) * s->H * s->B < (1 << 24) && ceil_div64(s->Nk, 64) * s->Hk * s->B < (1 << 24), "%s: more tiles than a launch takes", what);
    return 0;
}

Args args_of(const bndm_attention_shape *s, const void *q, const void *k, const void *v, const void *lam, const int32_t *q_start, const int32_t *kv_lengths) {
    Args a = {};
    a.q = q, a.k = k, a.v = v, a.lam = lam, a.q_start = q_start, a.kv_lengths = kv_lengths;
    a.Nq = s->Nq, a.Nk = s->Nk, a.B = (int)s->B, a.H = s->H, a.Hk = s->Hk, a.D = s->D, a.Dv = s->Dv, a.causal = s->causal != 0, a.lam_f32 = s->lam_f32, a.scale = s->scale;
    a.qb = s->q_strides[0], a.qn = s->q_strides[1], a.qh = s->q_strides[2];
    a.kb = s->k_strides[0], a.kn = s->k_strides[1], a.kh = s->k_strides[2];
    a.vb = s->v_strides[0], a.vn = s->v_strides[1], a.vh = s->v_strides[2];
    a.heads_per_row = 1, a.splits = 1, a.split_keys = s->Nk;
    return a;
}

bool aligned16(const void *p) { return (uint64_t)p % 16 == 0; }

}  // namespace
}  // namespace bndm

using namespace bndm;

extern "C" size_t bndm_tokens_attention_workspace_bytes(const bndm_attention_shape *s) {
    if (check("bndm_tokens_attention_workspace_bytes", s) || s->B == 0 || s->Nq == 0) return 0;
    const Plan p = plan_of(*s);
    return p.splits > 1 ? (size_t)s->B * s->H * s->Nq * p.splits * (2 * s->Dv + 4) * 4 : 0;
}

extern "C" int bndm_tokens_attention(const bndm_attention_shape *s, const void *q, const void *k, const void *v, const void *lam,
                                     const int32_t *q_start, const int32_t *kv_lengths, void *o, void *o2, float *lse, void *workspace,
                                     size_t workspace_bytes, void *stream) {
    if (int rc = check("bndm_tokens_attention", s)) return rc;
    if (s->B == 0 || s->Nq == 0) return 0;
    TOKENS_REQUIRE(q && lam && o && (s->Nk == 0 || (k && v)), "bndm_tokens_attention: NULL tensor");
    TOKENS_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(o2), "bndm_tokens_attention: tensors start at 16 bytes");
    TOKENS_REQUIRE((o2 == nullptr) == (lse == nullptr), "bndm_tokens_attention: o2 and lse go together");
    const Plan p = plan_of(*s);
    const size_t need = bndm_tokens_attention_workspace_bytes(s);
    TOKENS_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
                   "bndm_tokens_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    TOKENS_REQUIRE(p.blocks < (1 << 23), "bndm_tokens_attention: more tiles than a launch takes");
    Args a = args_of(s, q, k, v, lam, q_start, kv_lengths);
    a.o = o, a.o2 = o2, a.lse = lse;
    a.heads_per_row = p.heads_per_row, a.splits = p.splits, a.split_keys = p.split_keys;
    a.part = p.splits > 1 ? (float *)workspace : nullptr;
    const int d = padded(s->D, s->Dv);
    const hipStream_t st = (hipStream_t)stream;
    if (s->dtype == BNDM_DTYPE_F16) return d == 32 ? forward<f16, 32>(a, p, st) : d == 64 ? forward<f16, 64>(a, p, st) : forward<f16, 128>(a, p, st);
    return d == 32 ? forward<bf16, 32>(a, p, st) : d == 64 ? forward<bf16, 64>(a, p, st) : forward<bf16, 128>(a, p, st);
}

extern "C" size_t bndm_tokens_attention_backward_workspace_bytes(const bndm_attention_shape *s) {
    if (check("bndm_tokens_attention_backward_workspace_bytes", s)) return 0;
    return ((size_t)s->B * s->H * (2 * s->Nq + ceil_div64(s->Nq, 128) * 8) + s->B * s->Hk) * 4;
}

extern "C" int bndm_tokens_attention_backward(const bndm_attention_shape *s, const void *q, const void *k, const void *v, const void *lam,
                                              const int32_t *q_start, const int32_t *kv_lengths, const void *o, const void *o2, const float *lse,
                                              const void *dout, const int64_t dout_strides[3], void *dq, void *dk, void *dv, void *dlam,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check("bndm_tokens_attention_backward", s)) return rc;
    TOKENS_REQUIRE(s->B > 0 && s->Nq > 0, "bndm_tokens_attention_backward: no queries");
    TOKENS_REQUIRE(q && lam && o && o2 && lse && dout && dout_strides && dq && dlam && (s->Nk == 0 || (k && v && dk && dv)),
                   "bndm_tokens_attention_backward: NULL tensor");
    TOKENS_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(o2) && aligned16(dout) && aligned16(dq) && aligned16(dk) &&
                   aligned16(dv), "bndm_tokens_attention_backward: tensors start at 16 bytes");
    for (int i = 0; i < 3; ++i)
        TOKENS_REQUIRE(dout_strides[i] >= 0 && dout_strides[i] % 8 == 0 && (i != 1 || dout_strides[i] <= (1 << 23)),
                       "bndm_tokens_attention_backward: stride %lld: a multiple of 8, between tokens up to 2^23", (long long)dout_strides[i]);
    TOKENS_REQUIRE(s->H + s->B * s->Hk < (1 << 24), "bndm_tokens_attention_backward: more heads than a launch takes");
    const size_t need = bndm_tokens_attention_backward_workspace_bytes(s);
    TOKENS_REQUIRE(workspace && workspace_bytes >= need, "bndm_tokens_attention_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    Args a = args_of(s, q, k, v, lam, q_start, kv_lengths);
    a.o = (void *)o, a.o2 = (void *)o2, a.lse = (float *)lse;
    a.dout = dout, a.dob = dout_strides[0], a.don = dout_strides[1], a.doh = dout_strides[2];
    const int64_t runs = s->B * s->H * ceil_div64(s->Nq, 128) * 4;
    a.dq = dq, a.dk = dk, a.dv = dv, a.dlam = dlam;
    a.delta = (float *)workspace, a.d2_sums = a.delta + 2 * s->B * s->H * s->Nq, a.peaks = a.d2_sums + runs, a.steps = a.peaks + runs;
    const int d = padded(s->D, s->Dv);
    const hipStream_t st = (hipStream_t)stream;
    if (s->dtype == BNDM_DTYPE_F16) return d == 32 ? backward<f16, 32>(a, st) : d == 64 ? backward<f16, 64>(a, st) : backward<f16, 128>(a, st);
    return d == 32 ? backward<bf16, 32>(a, st) : d == 64 ? backward<bf16, 64>(a, st) : backward<bf16, 128>(a, st);
}
