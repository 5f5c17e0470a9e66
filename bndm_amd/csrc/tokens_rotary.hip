// Rotary positions on several axes.  Pair (a, b) of a head turns by the angle t = position[axis] * base^(-i / s):
//   a' = a cos t - b sin t,   b' = a sin t + b cos t;   the backward pass is the same with -t.
//
// Bound by memory: every element is read and written once, 3 operations each.  8 x 4096 tokens of 64 heads of 64 in f16 take 110 us
// (4.9 TB/s; a large copy moves 5.1), 2 x 20250 tokens of 32 heads of 96 in f32 178 us (5.6 TB/s).  A workgroup takes a run of tokens and forms their
// cosines and sines once, in LDS, for all heads of q and k; then its threads stream the heads in 16-byte pieces.  Angles are formed
// in 64 bits, as revolutions whose whole part is dropped before rounding to 32: position * frequency loses 2^-24 of a far position
// (0.06 radians at 10^6), which no later step can give back.
#include "tokens_common.hpp"
#include <cmath>

namespace bndm {
namespace {

constexpr int MAX_PAIRS = 128;
constexpr int THREADS = 256;

struct RotaryTable {
    double turns[MAX_PAIRS];      // frequency / (2 pi) of each pair
    uint8_t axis[MAX_PAIRS];
};

struct RotarySide {
    const void *in;
    void *out;
    int heads;
    int64_t sb, sn, sh;           // strides of `in`; `out` is contiguous
};

template <typename T, int V> struct Run { T v[V]; };

template <typename T, int V, bool WIDE> __device__ __forceinline__ Run<T, V> load_run(const T *p) {
    Run<T, V> r;
    if constexpr (WIDE && sizeof(T) * V == 16) *reinterpret_cast<u32x4 *>(&r) = *reinterpret_cast<const u32x4 *>(p);
    else if constexpr (WIDE && sizeof(T) * V == 8) *reinterpret_cast<u32x2 *>(&r) = *reinterpret_cast<const u32x2 *>(p);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = p[i];
    return r;
}
template <typename T, int V, bool WIDE> __device__ __forceinline__ void store_run(T *p, const Run<T, V> &r) {
    if constexpr (WIDE && sizeof(T) * V == 16) *reinterpret_cast<u32x4 *>(p) = *reinterpret_cast<const u32x4 *>(&r);
    else if constexpr (WIDE && sizeof(T) * V == 8) *reinterpret_cast<u32x2 *>(p) = *reinterpret_cast<const u32x2 *>(&r);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = r.v[i];
}

// V: elements of one piece, WIDE: read and written as one.  INTERLEAVED: a piece is V / 2 pairs; otherwise two pieces, D / 2 apart, are V pairs.
template <typename T, int V, bool WIDE, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotarySide q, RotarySide k, const void *positions, int position_type,
                                                         int64_t pb, int64_t pn, int64_t pa, int64_t tokens, int64_t N, int D,
                                                         int per_block, float sign, RotaryTable table) {
    extern __shared__ float2 turn[];                       // [per_block][D / 2]: cosine, sine
    const int half = D / 2;
    const int64_t t0 = (int64_t)blockIdx.x * per_block;
    const int nt = (int)min((int64_t)per_block, tokens - t0);

    for (int i = threadIdx.x; i < nt * half; i += THREADS) {
        const int t = i / half, j = i - t * half;
        const int64_t tok = t0 + t, b = tok / N, n = tok - b * N;
        const int64_t at = b * pb + n * pn + table.axis[j] * pa;
        const double p = position_type == 0 ? (double)((const int32_t *)positions)[at]
                       : position_type == 1 ? (double)((const int64_t *)positions)[at]
                                            : (double)((const float *)positions)[at];
        double r = p * table.turns[j];
        r -= rint(r);
        float s, c;
        sincospif(2.0f * (float)r, &s, &c);
        turn[i] = make_float2(c, sign * s);
    }
    __syncthreads();

    const int heads = q.heads + k.heads;
    const int pieces = INTERLEAVED ? D / V : half / V;     // work items of a head
    const int items = nt * heads * pieces;
#pragma unroll 2
    for (int i = threadIdx.x; i < items; i += THREADS) {
        const int th = i / pieces, c = i - th * pieces;
        const int t = th / heads, h = th - t * heads;
        const bool second = h >= q.heads;
        const int hh = second ? h - q.heads : h;
        const int64_t tok = t0 + t, b = tok / N, n = tok - b * N;
        const T *in = (const T *)(second ? k.in : q.in) + b * (second ? k.sb : q.sb) + n * (second ? k.sn : q.sn) +
                      hh * (second ? k.sh : q.sh) + c * V;
        T *out = (T *)(second ? k.out : q.out) + (tok * (second ? k.heads : q.heads) + hh) * D + c * V;
        if constexpr (INTERLEAVED) {
            const Run<T, V> x = load_run<T, V, WIDE>(in);
            Run<T, V> y;
            const float2 *cs = turn + t * half + c * (V / 2);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const float a = (float)x.v[2 * e], bb = (float)x.v[2 * e + 1];
                y.v[2 * e] = (T)(a * cs[e].x - bb * cs[e].y);
                y.v[2 * e + 1] = (T)(a * cs[e].y + bb * cs[e].x);
            }
            store_run<T, V, WIDE>(out, y);
        } else {
            const Run<T, V> x = load_run<T, V, WIDE>(in), w = load_run<T, V, WIDE>(in + half);
            Run<T, V> y, z;
            const float2 *cs = turn + t * half + c * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float a = (float)x.v[e], bb = (float)w.v[e];
                y.v[e] = (T)(a * cs[e].x - bb * cs[e].y);
                z.v[e] = (T)(a * cs[e].y + bb * cs[e].x);
            }
            store_run<T, V, WIDE>(out, y);
            store_run<T, V, WIDE>(out + half, z);
        }
    }
}

// elements of a piece: the widest of 16, 8 bytes or one pair that sizes, strides and addresses allow
int piece_of(const RotarySide &s, int run, int size) {
    int v = 16 / size;
    while (v > 1) {
        const uint64_t bytes = (uint64_t)v * size;
        if (run % v == 0 && s.sb % v == 0 && s.sn % v == 0 && s.sh % v == 0 && (uint64_t)s.in % bytes == 0 && (uint64_t)s.out % bytes == 0) break;
        v /= 2;
    }
    return v;
}

template <typename T, int V, bool WIDE, bool I>
int launch(const RotarySide &q, const RotarySide &k, const void *positions, int type, const int64_t *ps, int64_t B, int64_t N, int D,
            int sign, const RotaryTable &table, hipStream_t stream) {
    // tokens of a workgroup: about 8 pieces a thread, while 1024 workgroups (four for each CU) remain; 8 KB of LDS at most
    const int64_t tokens = B * N;
    const int pieces = (q.heads + k.heads) * (I ? D / V : D / 2 / V);
    int per = (int)min((int64_t)(1024 / (D / 2)), max((int64_t)1, (int64_t)8 * THREADS / max(1, pieces)));
    per = (int)max((int64_t)1, min((int64_t)per, tokens / 1024));
    const int64_t blocks = ceil_div64(tokens, per);
    TOKENS_REQUIRE(blocks < (1 << 24), "bndm_tokens_rotary: more tokens than a launch takes");
    hipLaunchKernelGGL((rotary_kernel<T, V, WIDE, I>), dim3((unsigned)blocks), dim3(THREADS), per * (D / 2) * sizeof(float2), stream,
                       q, k, positions, type, ps[0], ps[1], ps[2], tokens, N, D, per, sign ? -1.0f : 1.0f, table);
    return tokens_launch_status("rotary");
}

template <typename T>
int dispatch(const RotarySide &q, const RotarySide &k, const void *positions, int type, const int64_t *ps, int64_t B, int64_t N, int D,
              int interleaved, int inverse, const RotaryTable &table, hipStream_t stream) {
    const int run = interleaved ? D : D / 2;
    int v = piece_of(q, run, sizeof(T));
    if (k.heads) v = min(v, piece_of(k, run, sizeof(T)));
    if (interleaved) {
        if (v * sizeof(T) == 16) return launch<T, 16 / sizeof(T), true, true>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
        if (v * sizeof(T) == 8) return launch<T, 8 / sizeof(T), true, true>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
        return launch<T, 2, false, true>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
    }
    if (v * sizeof(T) == 16) return launch<T, 16 / sizeof(T), true, false>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
    if (v * sizeof(T) == 8) return launch<T, 8 / sizeof(T), true, false>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
    return launch<T, 1, false, false>(q, k, positions, type, ps, B, N, D, inverse, table, stream);
}

}  // namespace
}  // namespace bndm

using namespace bndm;

extern "C" int bndm_tokens_rotary(const void *q, const int64_t q_strides[3], void *q_out, int q_heads, const void *k,
                                  const int64_t k_strides[3], void *k_out, int k_heads, const void *positions,
                                  const int64_t position_strides[3], int position_type, int64_t B, int64_t N, int D,
                                  const int *sections, int axes, double base, int interleaved, int inverse, int dtype, void *stream) {
    TOKENS_REQUIRE(B >= 0 && N >= 0 && q_heads >= 0 && k_heads >= 0, "bndm_tokens_rotary: negative size");
    TOKENS_REQUIRE(D >= 2 && D % 2 == 0 && D <= 2 * MAX_PAIRS, "bndm_tokens_rotary: head size %d: an even number up to %d", D, 2 * MAX_PAIRS);
    TOKENS_REQUIRE(dtype == BNDM_DTYPE_F16 || dtype == BNDM_DTYPE_BF16 || dtype == BNDM_DTYPE_F32, "bndm_tokens_rotary: dtype %d", dtype);
    TOKENS_REQUIRE(position_type >= 0 && position_type <= 2, "bndm_tokens_rotary: position type %d", position_type);
    TOKENS_REQUIRE(sections && axes >= 1 && axes <= BNDM_TOKENS_MAX_AXES, "bndm_tokens_rotary: %d axes: 1 to %d", axes, BNDM_TOKENS_MAX_AXES);
    TOKENS_REQUIRE(std::isfinite(base) && base > 0.0, "bndm_tokens_rotary: base must be a positive number");
    RotaryTable table;
    int j = 0;
    for (int a = 0; a < axes; ++a) {
        TOKENS_REQUIRE(sections[a] >= 0 && sections[a] <= D / 2 - j, "bndm_tokens_rotary: sections must add up to half the head size, %d", D / 2);
        const double step = sections[a] ? pow(base, -1.0 / sections[a]) : 1.0;
        double f = 0.15915494309189533577;                 // 1 / (2 pi)
        for (int i = 0; i < sections[a]; ++i, ++j) {
            table.turns[j] = f;
            table.axis[j] = (uint8_t)a;
            f *= step;
        }
    }
    TOKENS_REQUIRE(j == D / 2, "bndm_tokens_rotary: sections must add up to half the head size, %d", D / 2);
    if (B == 0 || N == 0 || q_heads + k_heads == 0) return 0;
    TOKENS_REQUIRE(positions && position_strides && (!q_heads || (q && q_out && q_strides)) && (!k_heads || (k && k_out && k_strides)),
                   "bndm_tokens_rotary: NULL tensor");
    TOKENS_REQUIRE(B * N <= 0x7fffffff && (int64_t)(q_heads + k_heads) * D <= (1 << 22), "bndm_tokens_rotary: more tokens or heads than a launch takes");
    RotarySide sq = {q, q_out, q_heads, 0, 0, 0}, sk = {k, k_out, k_heads, 0, 0, 0};
    if (q_heads) sq.sb = q_strides[0], sq.sn = q_strides[1], sq.sh = q_strides[2];
    if (k_heads) sk.sb = k_strides[0], sk.sn = k_strides[1], sk.sh = k_strides[2];
    if (dtype == BNDM_DTYPE_F16) return dispatch<f16>(sq, sk, positions, position_type, position_strides, B, N, D, interleaved, inverse, table, (hipStream_t)stream);
    if (dtype == BNDM_DTYPE_BF16) return dispatch<bf16>(sq, sk, positions, position_type, position_strides, B, N, D, interleaved, inverse, table, (hipStream_t)stream);
    return dispatch<float>(sq, sk, positions, position_type, position_strides, B, N, D, interleaved, inverse, table, (hipStream_t)stream);
}
