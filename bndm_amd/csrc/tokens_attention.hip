// Differential attention  o = (P1 - lam P2) v,  P_m = softmax(scale q_m k_m^T), and its gradients, on the matrix units.
//
// Forward: one pass over the keys for both maps at once, with a running maximum and sum each; the scores are formed TRANSPOSED
// (keys down, queries across), so a lane holds one query: maxima and sums are over its own registers, its running statistics are
// scalars to it, and the weights of a step are at once the right operand of  o^T += v^T P^T.  v^T comes out of LDS by transposing
// reads, each fragment used for both maps.  For few queries the keys are split over workgroups and the parts joined by a second kernel.
//
// Backward, with dP = do v^T (the same for both maps), D_m = rowsum(P_m dP) = do . o_m:
//   dS1 = P1 (dP - D1),  dS2 = -lam P2 (dP - D2),  dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P1 - lam P2)^T do,
//   dlam = - sum over rows of D2.
// Two kernels, each with the sums it owns in registers: no atomics, and the same result every time.
//
// Statistics, sums and gradients' sums are 32 bits; weights (P, dS) are rounded to the inputs' type for the matrix units, as products
// of 16-bit operands are what those take.
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
};

// tile of `R` rows of `C` chunks at `base` (rows `stride` elements apart) into LDS; rows >= rows_in and chunks >= chunks_in are zeros.
// NW waves share the work; R * C is a multiple of 64 * NW
template <int R, int C, int NW>
__device__ __forceinline__ void stage_rows(char *lds, const void *base, int stride, int rows_in, int chunks_in, int w, int l) {
    const __amdgpu_buffer_rsrc_t rs = uniform_rsrc(base, kAnywhere);
#pragma unroll
    for (int i = 0; i < R * C / (64 * NW); ++i) {
        const int at = (i * NW + w) * 64 + l, row = at / C, c = (at % C) ^ swizzle<C>(row);
        const bool in = row < rows_in && c < chunks_in;
        const uint32_t off = in ? (uint32_t)(row * stride + c * 8) * 2u : kNowhere;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (i * NW + w) * 1024), 16, off, 0, 0, 0);
    }
}

// 8 values (chunk c) of row `row` of a tile
template <int C> __device__ __forceinline__ s16x8 row_fragment(const char *lds, int row, int c) {
    return *reinterpret_cast<const s16x8 *>(lds + row * (C * 16) + ((c ^ swizzle<C>(row)) << 4));
}

// operand whose rows are the tile's COLUMNS col0 .. + 31 and whose k are 16 of its rows, in the order in which a result tile holds
// them: lane half h has rows row0 + 4 h + {0..3} and row0 + 8 + 4 h + {0..3}
template <int C> __device__ __forceinline__ s16x8 column_fragment(const char *lds, int row0, int col0, int l) {
    const int i = l & 15, col = col0 + (l & 16) + 4 * (i & 3), row = row0 + 4 * (l >> 5) + (i >> 2);
    const s16x4 lo = lds_read_tr(lds + row * (C * 16) + (((col >> 3) ^ swizzle<C>(row)) << 4) + (col & 4) * 2);
    const s16x4 hi = lds_read_tr(lds + (row + 8) * (C * 16) + (((col >> 3) ^ swizzle<C>(row + 8)) << 4) + (col & 4) * 2);
    return join(lo, hi);
}

// registers 8 s .. 8 s + 7 of a result tile as an operand whose k are rows 16 s .. 16 s + 15 in that order
template <typename T> __device__ __forceinline__ s16x8 as_operand(const f32x16 &p, int s) {
    return pack8<T>(p[8 * s], p[8 * s + 1], p[8 * s + 2], p[8 * s + 3], p[8 * s + 4], p[8 * s + 5], p[8 * s + 6], p[8 * s + 7]);
}

__device__ __forceinline__ int tile_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

template <int N> __device__ __forceinline__ void clear(f32x16 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] = 0.f;
}

__device__ __forceinline__ float both_halves_max(float x) { return fmaxf(x, __shfl_xor(x, 32)); }
__device__ __forceinline__ float both_halves_sum(float x) { return x + __shfl_xor(x, 32); }

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
// NW waves, 32 rows (queries) each; KT keys a tile.  DT: head size rounded up to 32, 64, 128; values are up to 2 DT wide.
template <typename T, int DT, int NW, int KT>
__global__ __launch_bounds__(64 * NW) void attention_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT;
    constexpr int K_BYTES = KT * CK * 16, V_BYTES = KT * CV * 16, STAGE = 2 * K_BYTES + V_BYTES;
    __shared__ __attribute__((aligned(16))) char smem[2][STAGE];
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- which rows: (batch, group of query heads, tile of rows, part of the keys)
    const int64_t rows = a.Nq * a.heads_per_row;
    const int tiles = (int)((rows + 32 * NW - 1) / (32 * NW));
    int id = blockIdx.x;
    const int split = id % a.splits; id /= a.splits;
    const int tile = id % tiles; id /= tiles;
    const int groups = a.H / a.heads_per_row;
    const int group = id % groups, b = id / groups;
    const int hk = group * a.heads_per_row / (a.H / a.Hk);
    const int64_t row = (int64_t)tile * 32 * NW + w * 32 + (l & 31);
    const bool row_in = row < rows;
    const int sub = row_in ? (int)(row / a.Nq) : 0;
    const int64_t i = row_in ? row - (int64_t)sub * a.Nq : 0;
    const int head = group * a.heads_per_row + sub;

    const int64_t start = start_of(a, b), len = length_of(a, b);
    const int64_t sees = !row_in ? 0 : a.causal ? min(len, max((int64_t)0, start + i + 1)) : len;   // keys that this row sees
    // (rows of one head are in order; several heads in one tile: the last query's keys for all)
    int64_t most = len;
    if (a.causal) {
        const int64_t last = a.heads_per_row > 1 ? a.Nq - 1 : min(a.Nq - 1, (int64_t)(tile + 1) * 32 * NW - 1);
        most = min(len, max((int64_t)0, start + last + 1));
    }
    int64_t fewest = len;                                   // keys that every row of the wave sees
    if (a.causal) {
        const int64_t first = a.heads_per_row > 1 ? 0 : (int64_t)tile * 32 * NW + w * 32;
        fewest = min(len, max((int64_t)0, start + first + 1));
    }
    const int64_t j_begin = (int64_t)split * a.split_keys, j_end = min(most, j_begin + a.split_keys);

    // ---- queries: right operands, in registers
    s16x8 qf[2][DT / 16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const T *p = (const T *)a.q + (int64_t)b * a.qb + i * a.qn + (int64_t)(2 * head + m) * a.qh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            qf[m][s] = load8(p + c * 8, row_in && c * 8 < a.D);
        }
    }

    f32x16 acc[2][DV / 32];
    clear(acc[0]);
    clear(acc[1]);
    float top[2] = {kLowest, kLowest}, total[2] = {0.f, 0.f};
    const float to_log2 = a.scale * kLog2e;

    const T *kp[2] = {(const T *)a.k + (int64_t)b * a.kb + (int64_t)(2 * hk) * a.kh, nullptr};
    kp[1] = kp[0] + a.kh;
    const T *vp = (const T *)a.v + (int64_t)b * a.vb + (int64_t)hk * a.vh;
    auto fetch = [&](char *to, int64_t j) {
        const int in = (int)min((int64_t)KT, len - j);
        stage_rows<KT, CK, NW>(to, kp[0] + j * a.kn, (int)a.kn, in, a.D / 8, w, l);
        stage_rows<KT, CK, NW>(to + K_BYTES, kp[1] + j * a.kn, (int)a.kn, in, a.D / 8, w, l);
        stage_rows<KT, CV, NW>(to + 2 * K_BYTES, vp + j * a.vn, (int)a.vn, in, a.Dv / 8, w, l);
    };

    if (j_begin < j_end) fetch(smem[0], j_begin);
    int buf = 0;
    for (int64_t j = j_begin; j < j_end; j += KT, buf ^= 1) {
        wait_lds_dma();
        __syncthreads();
        if (j + KT < j_end) fetch(smem[buf ^ 1], j + KT);
        const char *ks = smem[buf], *vs = ks + 2 * K_BYTES;
        const bool masked = j + KT > fewest;

        s16x8 pf[2][KT / 16];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x16 s[KT / 32];
            clear(s);
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int d = 0; d < DT / 16; ++d)
                    s[t] = mfma32<T>(row_fragment<CK>(ks + m * K_BYTES, 32 * t + (l & 31), 2 * d + h32), qf[m][d], s[t]);
            if (masked) {
                const int n = (int)min((int64_t)KT, max((int64_t)0, sees - j));
#pragma unroll
                for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * t + tile_row(r, h32) >= n) s[t][r] = -INFINITY;
            }
            float high = s[0][0];
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) high = fmaxf(high, s[t][r]);
            high = both_halves_max(high) * to_log2;
            const float next = fmaxf(top[m], high);
            const float shrink = __builtin_amdgcn_exp2f(top[m] - next);
            top[m] = next;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], to_log2, -next));
                    sum += s[t][r];
                }
            total[m] = total[m] * shrink + sum;
#pragma unroll
            for (int t = 0; t < DV / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[m][t][r] *= shrink;
#pragma unroll
            for (int t = 0; t < KT / 16; ++t) pf[m][t] = as_operand<T>(s[t / 2], t & 1);
        }
#pragma unroll
        for (int t = 0; t < DV / 32; ++t)
#pragma unroll
            for (int s = 0; s < KT / 16; ++s) {
                const s16x8 vf = column_fragment<CV>(vs, 16 * s, 32 * t, l);
                acc[0][t] = mfma32<T>(vf, pf[0][s], acc[0][t]);
                acc[1][t] = mfma32<T>(vf, pf[1][s], acc[1][t]);
            }
    }
    total[0] = both_halves_sum(total[0]);
    total[1] = both_halves_sum(total[1]);
    if (!row_in) return;

    if (a.part) {                                           // unfinished sums of this part
        float *to = a.part + ((((int64_t)b * a.H + head) * a.Nq + i) * a.splits + split) * (2 * a.Dv + 4);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < DV / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int d = 32 * t + tile_row(r, h32);
                    const f32x4 v = {acc[m][t][r], acc[m][t][r + 1], acc[m][t][r + 2], acc[m][t][r + 3]};
                    if (d < a.Dv) *reinterpret_cast<f32x4 *>(to + m * a.Dv + d) = v;
                }
        if (h32 == 0) *reinterpret_cast<f32x4 *>(to + 2 * a.Dv) = (f32x4){top[0], top[1], total[0], total[1]};
        return;
    }
    const float lam = lam_of<T>(a, head);
    const float w1 = total[0] == 0.f ? 0.f : 1.0f / total[0], w2 = total[1] == 0.f ? 0.f : 1.0f / total[1];
    const int64_t at = (((int64_t)b * a.Nq + i) * a.H + head) * a.Dv;
#pragma unroll
    for (int t = 0; t < DV / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * t + tile_row(r, h32);
            if (d < a.Dv) {
                float x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[e] = acc[1][t][r + e] * w2;
                    x[e] = acc[0][t][r + e] * w1 - lam * y[e];
                }
                *reinterpret_cast<s16x4 *>((T *)a.o + at + d) = pack4<T>(x[0], x[1], x[2], x[3]);
                if (a.o2) *reinterpret_cast<s16x4 *>((T *)a.o2 + at + d) = pack4<T>(y[0], y[1], y[2], y[3]);
            }
        }
    if (a.lse && h32 == 0)
#pragma unroll
        for (int m = 0; m < 2; ++m)
            a.lse[((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i] = total[m] == 0.f ? INFINITY : top[m] + __log2f(total[m]);
}

// joins the parts of a row: one wave a row, each lane every 64th value
template <typename T> __global__ __launch_bounds__(256) void attention_join_kernel(Args a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    if (row >= (int64_t)a.B * a.H * a.Nq) return;
    const int width = 2 * a.Dv + 4;
    const float *p = a.part + row * a.splits * width;
    float top[2] = {kLowest, kLowest}, total[2] = {0.f, 0.f};
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
        for (int m = 0; m < 2; ++m) top[m] = fmaxf(top[m], p[(int64_t)s * width + 2 * a.Dv + m]);
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
        for (int m = 0; m < 2; ++m)
            total[m] += p[(int64_t)s * width + 2 * a.Dv + 2 + m] * __builtin_amdgcn_exp2f(p[(int64_t)s * width + 2 * a.Dv + m] - top[m]);
    const float w[2] = {total[0] == 0.f ? 0.f : 1.0f / total[0], total[1] == 0.f ? 0.f : 1.0f / total[1]};
    const int64_t i = row % a.Nq, bh = row / a.Nq;
    const int head = (int)(bh % a.H);
    const int64_t b = bh / a.H;
    const float lam = lam_of<T>(a, head);
    const int64_t at = ((b * a.Nq + i) * a.H + head) * a.Dv;
    for (int d = l; d < a.Dv; d += 64) {
        float x[2] = {0.f, 0.f};
        for (int s = 0; s < a.splits; ++s)
#pragma unroll
            for (int m = 0; m < 2; ++m)
                x[m] += p[(int64_t)s * width + m * a.Dv + d] * __builtin_amdgcn_exp2f(p[(int64_t)s * width + 2 * a.Dv + m] - top[m]);
        ((T *)a.o)[at + d] = (T)(x[0] * w[0] - lam * (x[1] * w[1]));
        if (a.o2) ((T *)a.o2)[at + d] = (T)(x[1] * w[1]);
    }
    if (a.lse && l < 2) {
        const float t = l ? total[1] : total[0], m = l ? top[1] : top[0];
        a.lse[(b * 2 * a.H + 2 * head + l) * a.Nq + i] = t == 0.f ? INFINITY : m + __log2f(t);
    }
}

// ---------------------------------------------------------------------------------------------- gradients of the queries
// As the forward pass: a lane holds one query, dS^T is at once the right operand of  dq^T += k^T dS^T.  Also D1, D2 for the next kernel.
template <typename T, int DT, int KT>
__global__ __launch_bounds__(THREADS) void attention_dq_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 4;
    constexpr int K_BYTES = KT * CK * 16, V_BYTES = KT * CV * 16, STAGE = 2 * K_BYTES + V_BYTES;
    __shared__ __attribute__((aligned(16))) char smem[2][STAGE];
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)((a.Nq + 127) / 128);
    int id = blockIdx.x;
    const int tile = id % tiles; id /= tiles;
    const int head = id % a.H, b = id / a.H;
    const int hk = head / (a.H / a.Hk);
    const int64_t row = (int64_t)tile * 128 + w * 32 + (l & 31);
    const bool row_in = row < a.Nq;
    const int64_t i = row_in ? row : 0;
    const int64_t start = start_of(a, b), len = length_of(a, b);
    const int64_t sees = !row_in ? 0 : a.causal ? min(len, max((int64_t)0, start + i + 1)) : len;
    int64_t j_end = len, fewest = len;
    if (a.causal) {
        j_end = min(len, max((int64_t)0, start + min(a.Nq, (int64_t)(tile + 1) * 128)));
        fewest = min(len, max((int64_t)0, start + (int64_t)tile * 128 + w * 32 + 1));
    }

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
    // D2 = do . o2, D1 = do . (o + lam o2)
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
        delta[0] += lam * delta[1];
    }
    float lse[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int64_t at = ((int64_t)b * 2 * a.H + 2 * head + m) * a.Nq + i;
        lse[m] = row_in ? a.lse[at] : INFINITY;
        if (row_in && h32 == 0) a.delta[at] = delta[m];
    }

    f32x16 acc[2][DT / 32];
    clear(acc[0]);
    clear(acc[1]);
    const float to_log2 = a.scale * kLog2e;
    const T *kp[2] = {(const T *)a.k + (int64_t)b * a.kb + (int64_t)(2 * hk) * a.kh, nullptr};
    kp[1] = kp[0] + a.kh;
    const T *vp = (const T *)a.v + (int64_t)b * a.vb + (int64_t)hk * a.vh;
    auto fetch = [&](char *to, int64_t j) {
        const int in = (int)min((int64_t)KT, len - j);
        stage_rows<KT, CK, NW>(to, kp[0] + j * a.kn, (int)a.kn, in, a.D / 8, w, l);
        stage_rows<KT, CK, NW>(to + K_BYTES, kp[1] + j * a.kn, (int)a.kn, in, a.D / 8, w, l);
        stage_rows<KT, CV, NW>(to + 2 * K_BYTES, vp + j * a.vn, (int)a.vn, in, a.Dv / 8, w, l);
    };
    if (0 < j_end) fetch(smem[0], 0);
    int buf = 0;
    for (int64_t j = 0; j < j_end; j += KT, buf ^= 1) {
        wait_lds_dma();
        __syncthreads();
        if (j + KT < j_end) fetch(smem[buf ^ 1], j + KT);
        const char *ks = smem[buf], *vs = ks + 2 * K_BYTES;
        const bool masked = j + KT > fewest || sees == 1;
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
            f32x16 dp[1], s[1];
            clear(dp);
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) dp[0] = mfma32<T>(row_fragment<CV>(vs, 32 * t + (l & 31), 2 * d + h32), gf[d], dp[0]);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                clear(s);
#pragma unroll
                for (int d = 0; d < DT / 16; ++d)
                    s[0] = mfma32<T>(row_fragment<CK>(ks + m * K_BYTES, 32 * t + (l & 31), 2 * d + h32), qf[m][d], s[0]);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], to_log2, -lse[m])) * (dp[0][r] - delta[m]);
                if (masked) {                               // (a row that sees one key has weight 1 there whatever its score)
                    const int n = sees == 1 ? 0 : (int)min((int64_t)KT, max((int64_t)0, sees - j));
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * t + tile_row(r, h32) >= n) s[0][r] = 0.f;
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const s16x8 ds = as_operand<T>(s[0], g);
#pragma unroll
                    for (int d = 0; d < DT / 32; ++d)
                        acc[m][d] = mfma32<T>(column_fragment<CK>(ks + m * K_BYTES, 32 * t + 16 * g, 32 * d, l), ds, acc[m][d]);
                }
            }
        }
    }
    if (!row_in) return;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float f = m ? -lam * a.scale : a.scale;
        T *to = (T *)a.dq + (((int64_t)b * a.Nq + i) * 2 * a.H + 2 * head + m) * a.D;
#pragma unroll
        for (int t = 0; t < DT / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * t + tile_row(r, h32);
                if (d < a.D)
                    *reinterpret_cast<s16x4 *>(to + d) = pack4<T>(acc[m][t][r] * f, acc[m][t][r + 1] * f, acc[m][t][r + 2] * f, acc[m][t][r + 3] * f);
            }
    }
}

// ---------------------------------------------------------------------------------------------- gradients of keys and values
// The other way round: a lane holds one key, scores have queries down and keys across, W = P1 - lam P2 and dS_m are the right operands
// of  dv^T += do^T W  and  dk_m^T += q_m^T dS_m.  Keys and values of 128 rows stay in registers while the queries of every head that
// reads them pass through LDS, so shared heads' gradients are summed here.
template <typename T, int DT, int QT>
__global__ __launch_bounds__(THREADS) void attention_dkv_kernel(Args a) {
    constexpr int CK = DT / 8, CV = DT / 4, DV = 2 * DT, NW = 4;
    constexpr int Q_BYTES = QT * CK * 16, G_BYTES = QT * CV * 16, STAGE = 2 * Q_BYTES + G_BYTES;
    __shared__ __attribute__((aligned(16))) char smem[2][STAGE];
    __shared__ __attribute__((aligned(16))) float stats[2][4][QT];     // lse1, lse2, D1, D2 of the queries of a tile
    const int tid = threadIdx.x, l = tid & 63, h32 = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)((a.Nk + 127) / 128);
    int id = blockIdx.x;
    const int tile = id % tiles; id /= tiles;
    const int hk = id % a.Hk, b = id / a.Hk;
    const int per = a.H / a.Hk;
    const int64_t start = start_of(a, b), len = length_of(a, b);
    const int64_t key0 = (int64_t)tile * 128 + w * 32, key = key0 + (l & 31);
    const bool key_in = key < len;

    s16x8 kf[2][DT / 16], vf[DV / 16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const T *p = (const T *)a.k + (int64_t)b * a.kb + (key_in ? key : 0) * a.kn + (int64_t)(2 * hk + m) * a.kh;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const int c = 2 * s + h32;
            kf[m][s] = load8(p + c * 8, key_in && c * 8 < a.D);
        }
    }
    {
        const T *p = (const T *)a.v + (int64_t)b * a.vb + (key_in ? key : 0) * a.vn + (int64_t)hk * a.vh;
#pragma unroll
        for (int s = 0; s < DV / 16; ++s) {
            const int c = 2 * s + h32;
            vf[s] = load8(p + c * 8, key_in && c * 8 < a.Dv);
        }
    }
    f32x16 dk[2][DT / 32], dv[DV / 32];
    clear(dk[0]);
    clear(dk[1]);
    clear(dv);
    const float to_log2 = a.scale * kLog2e;

    // queries that see any key of this workgroup
    int64_t i_begin = 0;
    if (a.causal) i_begin = max((int64_t)0, (int64_t)tile * 128 - start) / QT * QT;
    if ((int64_t)tile * 128 >= len) i_begin = a.Nq;
    const int64_t i_first = i_begin;
    const int per_head = i_first < a.Nq ? (int)((a.Nq - i_first + QT - 1) / QT) : 0;
    const int steps = per_head * per;

    auto fetch = [&](int to, int step) {
        const int g = step / per_head;
        const int64_t i = i_first + (int64_t)(step - g * per_head) * QT;
        const int head = hk * per + g, in = (int)min((int64_t)QT, a.Nq - i);
        const T *qp = (const T *)a.q + (int64_t)b * a.qb + i * a.qn + (int64_t)(2 * head) * a.qh;
        stage_rows<QT, CK, NW>(smem[to], qp, (int)a.qn, in, a.D / 8, w, l);
        stage_rows<QT, CK, NW>(smem[to] + Q_BYTES, qp + a.qh, (int)a.qn, in, a.D / 8, w, l);
        stage_rows<QT, CV, NW>(smem[to] + 2 * Q_BYTES, (const T *)a.dout + (int64_t)b * a.dob + i * a.don + (int64_t)head * a.doh, (int)a.don, in,
                               a.Dv / 8, w, l);
        // (queries past the end: P = exp2(s - inf) = 0)
        for (int e = tid; e < 4 * QT; e += THREADS) {
            const int what = e / QT, r = e % QT;
            const float *from = (what < 2 ? a.lse : a.delta) + ((int64_t)b * 2 * a.H + 2 * head + (what & 1)) * a.Nq + i;
            stats[to][what][r] = r < in ? from[r] : what < 2 ? INFINITY : 0.f;
        }
    };
    if (steps) fetch(0, 0);
    for (int step = 0; step < steps; ++step) {
        const int buf = step & 1;
        wait_lds_dma();
        __syncthreads();
        if (step + 1 < steps) fetch(buf ^ 1, step + 1);
        const int g = step / per_head;
        const int64_t i0 = i_first + (int64_t)(step - g * per_head) * QT;
        const float lam = lam_of<T>(a, hk * per + g);
        const char *qs = smem[buf], *gs = qs + 2 * Q_BYTES;
#pragma unroll
        for (int t = 0; t < QT / 32; ++t) {
            const int64_t it = i0 + 32 * t;
            // some pair is hidden, or some row sees one key only
            const bool masked = key0 + 32 > len || (a.causal && key0 + 31 > start + it) || len == 1 || (a.causal && start + it <= 0);
            f32x16 dp[1], s[1], wt;
            clear(dp);
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) dp[0] = mfma32<T>(row_fragment<CV>(gs, 32 * t + (l & 31), 2 * d + h32), vf[d], dp[0]);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                clear(s);
#pragma unroll
                for (int d = 0; d < DT / 16; ++d)
                    s[0] = mfma32<T>(row_fragment<CK>(qs + m * Q_BYTES, 32 * t + (l & 31), 2 * d + h32), kf[m][d], s[0]);
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 ls = *reinterpret_cast<const f32x4 *>(&stats[buf][m][32 * t + tile_row(r, h32)]);
                    const f32x4 de = *reinterpret_cast<const f32x4 *>(&stats[buf][2 + m][32 * t + tile_row(r, h32)]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r + e], to_log2, -ls[e]));
                        float ds = p * (dp[0][r + e] - de[e]);
                        if (masked) {
                            const int64_t last = start + it + tile_row(r + e, h32);     // the last key that this query sees
                            if (key >= len || (a.causal && key > last)) p = ds = 0.f;
                            if (len == 1 || (a.causal && last == 0)) ds = 0.f;
                        }
                        if (m == 0) wt[r + e] = p;
                        else {
                            wt[r + e] -= lam * p;
                            ds *= -lam;
                        }
                        s[0][r + e] = ds;
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const s16x8 ds = as_operand<T>(s[0], x);
#pragma unroll
                    for (int d = 0; d < DT / 32; ++d)
                        dk[m][d] = mfma32<T>(column_fragment<CK>(qs + m * Q_BYTES, 32 * t + 16 * x, 32 * d, l), ds, dk[m][d]);
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const s16x8 wf = as_operand<T>(wt, x);
#pragma unroll
                for (int d = 0; d < DV / 32; ++d) dv[d] = mfma32<T>(column_fragment<CV>(gs, 32 * t + 16 * x, 32 * d, l), wf, dv[d]);
            }
        }
    }
    if (key >= a.Nk) return;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        T *to = (T *)a.dk + (((int64_t)b * a.Nk + key) * 2 * a.Hk + 2 * hk + m) * a.D;
#pragma unroll
        for (int t = 0; t < DT / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * t + tile_row(r, h32);
                if (d < a.D)
                    *reinterpret_cast<s16x4 *>(to + d) = pack4<T>(dk[m][t][r] * a.scale, dk[m][t][r + 1] * a.scale, dk[m][t][r + 2] * a.scale, dk[m][t][r + 3] * a.scale);
            }
    }
    T *to = (T *)a.dv + (((int64_t)b * a.Nk + key) * a.Hk + hk) * a.Dv;
#pragma unroll
    for (int t = 0; t < DV / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * t + tile_row(r, h32);
            if (d < a.Dv) *reinterpret_cast<s16x4 *>(to + d) = pack4<T>(dv[t][r], dv[t][r + 1], dv[t][r + 2], dv[t][r + 3]);
        }
}

// dlam[h] = - sum over sequences and queries of D2: one workgroup a head, in a fixed order
template <typename T> __global__ __launch_bounds__(THREADS) void attention_dlam_kernel(Args a) {
    __shared__ float part[THREADS];
    const int head = blockIdx.x;
    float sum = 0.f;
    for (int b = 0; b < a.B; ++b) {
        const float *d2 = a.delta + ((int64_t)b * 2 * a.H + 2 * head + 1) * a.Nq;
        for (int64_t i = threadIdx.x; i < a.Nq; i += THREADS) sum += d2[i];
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int n = THREADS / 2; n > 0; n /= 2) {
        if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (a.lam_f32) ((float *)a.dlam)[head] = -part[0];
        else ((T *)a.dlam)[head] = (T)(-part[0]);
    }
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
    // parts of the keys: as many as fill 256 CUs with four one-wave workgroups or one of four waves, of 256 keys at least
    const int64_t want = p.waves == 1 ? 1024 : 256;
    int64_t splits = tiles >= want ? 1 : ceil_div64(want, tiles);
    const int64_t most = s.Nk / 256 < 1 ? 1 : s.Nk / 256;
    if (splits > most) splits = most;
    p.split_keys = ceil_div64(ceil_div64(s.Nk, splits), 64) * 64;
    if (p.split_keys < 64) p.split_keys = 64;
    p.splits = (int)ceil_div64(s.Nk > 0 ? s.Nk : 1, p.split_keys);
    p.blocks = tiles * p.splits;
    return p;
}

template <typename T, int DT> int forward(const Args &a, const Plan &p, hipStream_t stream) {
    constexpr int KT = DT == 128 ? 32 : 64;
    if (p.waves == 1) hipLaunchKernelGGL((attention_kernel<T, DT, 1, 32>), dim3((unsigned)p.blocks), dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((attention_kernel<T, DT, 4, KT>), dim3((unsigned)p.blocks), dim3(256), 0, stream, a);
    if (int rc = tokens_launch_status("attention")) return rc;
    if (a.part) {
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)ceil_div64((int64_t)a.B * a.H * a.Nq, 4)), dim3(256), 0, stream, a);
        return tokens_launch_status("attention join");
    }
    return 0;
}

template <typename T, int DT> int backward(const Args &a, hipStream_t stream) {
    constexpr int KT = DT == 128 ? 32 : 64;
    const int64_t nq = ceil_div64(a.Nq, 128) * a.H * a.B, nk = ceil_div64(a.Nk, 128) * a.Hk * a.B;
    hipLaunchKernelGGL((attention_dq_kernel<T, DT, KT>), dim3((unsigned)nq), dim3(THREADS), 0, stream, a);
    if (int rc = tokens_launch_status("attention dq")) return rc;
    if (nk) {
        hipLaunchKernelGGL((attention_dkv_kernel<T, DT, KT>), dim3((unsigned)nk), dim3(THREADS), 0, stream, a);
        if (int rc = tokens_launch_status("attention dkv")) return rc;
    }
    hipLaunchKernelGGL((attention_dlam_kernel<T>), dim3(a.H), dim3(THREADS), 0, stream, a);
    return tokens_launch_status("attention dlam");
}

int check(const char *what, const bndm_attention_shape *s) {
    TOKENS_REQUIRE(s, "%s: NULL shape", what);
    TOKENS_REQUIRE(s->B >= 0 && s->Nq >= 0 && s->Nk >= 0 && s->B <= (1 << 20) && s->Nq <= (1 << 30) && s->Nk <= (1 << 30), "%s: sizes", what);
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
    TOKENS_REQUIRE(ceil_div64(s->Nq, 32) * s->H * s->B < (1 << 24) && ceil_div64(s->Nk, 128) * s->Hk * s->B < (1 << 24), "%s: more tiles than a launch takes", what);
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
    TOKENS_REQUIRE(p.blocks < (1 << 24), "bndm_tokens_attention: more tiles than a launch takes");
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
    return (size_t)s->B * 2 * s->H * s->Nq * 4;
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
    const size_t need = bndm_tokens_attention_backward_workspace_bytes(s);
    TOKENS_REQUIRE(workspace && workspace_bytes >= need, "bndm_tokens_attention_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    Args a = args_of(s, q, k, v, lam, q_start, kv_lengths);
    a.o = (void *)o, a.o2 = (void *)o2, a.lse = (float *)lse;
    a.dout = dout, a.dob = dout_strides[0], a.don = dout_strides[1], a.doh = dout_strides[2];
    a.dq = dq, a.dk = dk, a.dv = dv, a.dlam = dlam, a.delta = (float *)workspace;
    const int d = padded(s->D, s->Dv);
    const hipStream_t st = (hipStream_t)stream;
    if (s->dtype == BNDM_DTYPE_F16) return d == 32 ? backward<f16, 32>(a, st) : d == 64 ? backward<f16, 64>(a, st) : backward<f16, 128>(a, st);
    return d == 32 ? backward<bf16, 32>(a, st) : d == 64 ? backward<bf16, 64>(a, st) : backward<bf16, 128>(a, st);
}
