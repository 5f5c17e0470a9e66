// Linear layer y = act(x W^T + b) + r and its gradients, on the matrix units.
//
//   forward   y[m][n]  = sum_k x[m][k] W[n][k]        both operands hold the summed index along their rows
//   dx        dx[m][k] = sum_n dz[m][n] W[n][k]       the second holds it across its rows
//   dW        dW[n][k] = sum_m dz[m][n] x[m][k]       both hold it across their rows
//
// One kernel takes all three: an operand whose rows run along the summed index is read from LDS as rows, one whose rows run across it
// by transposing LDS reads, so no operand is copied into another layout first.
#include "tokens_common.hpp"

namespace bndm {
namespace {

// ---------------------------------------------------------------------------------------------- activation
// Phi(z): erfcf's error is relative, which 1 + erf(z) loses for negative z
__device__ __forceinline__ float act_value(int act, float z) {
    if (act == BNDM_ACT_SILU) return z / (1.0f + __expf(-z));
    if (act == BNDM_ACT_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);
    return z;
}
__device__ __forceinline__ float act_slope(int act, float z) {
    if (act == BNDM_ACT_SILU) {
        const float s = 1.0f / (1.0f + __expf(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    return 0.5f * erfcf(-0.70710678118654752f * z) + 0.39894228040143268f * z * __expf(-0.5f * z * z);
}

// ---------------------------------------------------------------------------------------------- the product
// C[m][n] = sum_k A(m, k) B(n, k).  TA false: A(m, k) = a[m * lda + k]; true: a[k * lda + m]; TB likewise.
// The B operand's index runs down the registers of a result tile, so a lane holds 4 consecutive n of one row m.
struct Epilogue {
    const void *bias;
    const void *residual;
    int64_t ldr;
    void *z;
    int act;
};

constexpr int BM = 128, BN = 128, BK = 64;
constexpr int NT = 256;

template <typename T> __device__ __forceinline__ void store_row4(const Epilogue &e, T *c, int64_t ldc, int64_t m, int64_t n, int64_t M, int64_t N,
                                                                 f32x4 v, bool wide) {
    if (m >= M || n >= N) return;
    const int left = (int)min((int64_t)4, N - n);
    float bias[4] = {0.f, 0.f, 0.f, 0.f}, res[4] = {0.f, 0.f, 0.f, 0.f};
    if (wide) {                                            // n % 4 == 0, N % 4 == 0, rows of 8-byte pieces
        if (e.bias) {
            const s16x4 b = *reinterpret_cast<const s16x4 *>((const T *)e.bias + n);
#pragma unroll
            for (int i = 0; i < 4; ++i) { const short s = b[i]; bias[i] = widen<T>(s); }
        }
        if (e.residual) {
            const s16x4 r = *reinterpret_cast<const s16x4 *>((const T *)e.residual + m * e.ldr + n);
#pragma unroll
            for (int i = 0; i < 4; ++i) { const short s = r[i]; res[i] = widen<T>(s); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) {
                if (e.bias) bias[i] = (float)((const T *)e.bias)[n + i];
                if (e.residual) res[i] = (float)((const T *)e.residual)[m * e.ldr + n + i];
            }
    }
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] += bias[i];
        y[i] = act_value(e.act, v[i]) + res[i];
    }
    if (wide) {
        if (e.z) *reinterpret_cast<s16x4 *>((T *)e.z + m * N + n) = pack4<T>(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<s16x4 *>(c + m * ldc + n) = pack4<T>(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) {
                if (e.z) ((T *)e.z)[m * N + n + i] = (T)v[i];
                c[m * ldc + n + i] = (T)y[i];
            }
    }
}

// one operand's tile of 128 rows x 64 of the summed index, 16 KB, in 16-byte chunks whose places are swizzled
//   rows along the summed index: [128][8 chunks];  across it: [64][16 chunks]
template <typename T, bool TR, bool WIDE>
__device__ __forceinline__ void stage(char *lds, const T *p, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t K, int tid) {
    constexpr int C = TR ? 16 : 8;
    const int64_t outer0 = TR ? k0 : row0, inner0 = TR ? row0 : k0;
    const int64_t outers = (TR ? K : rows) - outer0, inners = (TR ? rows : K) - inner0;   // what is there, from here on
    const T *base = p + outer0 * ld + inner0;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    if constexpr (WIDE) {
        const __amdgpu_buffer_rsrc_t rs = uniform_rsrc(base, kAnywhere);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = i * NT + tid, row = at / C, c = (at % C) ^ swizzle<C>(row);
            // (the inner extent is a multiple of 8 here, so a chunk is in or out as a whole)
            const bool in = row < outers && c * 8 < inners;
            const uint32_t off = in ? (uint32_t)(row * (int)ld + c * 8) * 2u : kNowhere;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (i * NT + w * 64) * 16), 16, off, 0, 0, 0);
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const int at = i * NT + tid, row = at / C, c = (at % C) ^ swizzle<C>(row);
            s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
            if (row < outers) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c * 8 + e < inners) v[e] = reinterpret_cast<const short *>(base)[row * ld + c * 8 + e];
            }
            *reinterpret_cast<s16x8 *>(lds + at * 16) = v;
        }
    }
}

// lane's 8 values of row `row` (of 32, + row0) and k = 16 s + 8 (l / 32) .. + 7
template <bool TR> __device__ __forceinline__ s16x8 fragment(const char *lds, int row0, int s, int l) {
    const int h = l >> 5;
    if constexpr (!TR) {
        const int row = row0 + (l & 31), c = 2 * s + h;
        return *reinterpret_cast<const s16x8 *>(lds + row * 128 + ((c ^ swizzle<8>(row)) << 4));
    } else {
        const int i = l & 15, col = row0 + (l & 16) + 4 * (i & 3);
        const int k = 16 * s + 8 * h + (i >> 2);
        const s16x4 lo = lds_read_tr(lds + k * 256 + (((col >> 3) ^ swizzle<16>(k)) << 4) + (col & 4) * 2);
        const s16x4 hi = lds_read_tr(lds + (k + 4) * 256 + (((col >> 3) ^ swizzle<16>(k + 4)) << 4) + (col & 4) * 2);
        return join(lo, hi);
    }
}

template <typename T, bool TA, bool TB, bool WIDE>
__global__ __launch_bounds__(NT) void gemm_kernel(const T *a, int64_t lda, const T *b, int64_t ldb, T *c, int64_t ldc, int64_t M, int64_t N,
                                                  int64_t K, Epilogue ep, int wide_out) {
    __shared__ __attribute__((aligned(16))) char smem[2][2 * BM * BK * 2];
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tiles_n = (unsigned)((N + BN - 1) / BN);
    const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * BM, n0 = (int64_t)(blockIdx.x % tiles_n) * BN;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int steps = (int)((K + BK - 1) / BK);
    if (steps) {
        stage<T, TA, WIDE>(smem[0], a, lda, m0, M, 0, K, tid);
        stage<T, TB, WIDE>(smem[0] + BM * BK * 2, b, ldb, n0, N, 0, K, tid);
    }
    for (int s = 0; s < steps; ++s) {
        wait_lds_dma();
        __syncthreads();                                   // tile s is there, and tile s - 1 has been read by every wave
        if (s + 1 < steps) {
            stage<T, TA, WIDE>(smem[(s + 1) & 1], a, lda, m0, M, (int64_t)(s + 1) * BK, K, tid);
            stage<T, TB, WIDE>(smem[(s + 1) & 1] + BM * BK * 2, b, ldb, n0, N, (int64_t)(s + 1) * BK, K, tid);
        }
        const char *ta = smem[s & 1], *tb = ta + BM * BK * 2;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
            s16x8 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = fragment<TA>(ta, wm + 32 * i, kk, l);
                fb[i] = fragment<TB>(tb, wn + 32 * i, kk, l);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma32<T>(fb[j], fa[i], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 v = {acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
                store_row4<T>(ep, c, ldc, m0 + wm + 32 * i + (l & 31), n0 + wn + 32 * j + 8 * r + 4 * (l >> 5), M, N, v, wide_out);
            }
}

template <typename T, bool TA, bool TB>
int gemm(const void *a, int64_t lda, const void *b, int64_t ldb, void *c, int64_t ldc, int64_t M, int64_t N, int64_t K, const Epilogue &ep,
         hipStream_t stream) {
    // 16-byte loads: rows and the index along them in pieces of 8 elements (a piece is inside or outside as a whole)
    const bool wide_in = lda % 8 == 0 && ldb % 8 == 0 && (uint64_t)a % 16 == 0 && (uint64_t)b % 16 == 0 && (TA ? M : K) % 8 == 0 &&
                         (TB ? N : K) % 8 == 0;
    const bool wide_out = N % 4 == 0 && ldc % 4 == 0 && (uint64_t)c % 8 == 0 && (!ep.bias || (uint64_t)ep.bias % 8 == 0) &&
                          (!ep.residual || ((uint64_t)ep.residual % 8 == 0 && ep.ldr % 4 == 0)) && (!ep.z || (uint64_t)ep.z % 8 == 0);
    const int64_t tiles = ceil_div64(N, BN) * ceil_div64(M, BM);
    TOKENS_REQUIRE(tiles < (1 << 24), "linear: more tiles than a launch takes");
    const dim3 grid((unsigned)tiles);
    if (wide_in) hipLaunchKernelGGL((gemm_kernel<T, TA, TB, true>), grid, dim3(NT), 0, stream, (const T *)a, lda, (const T *)b, ldb, (T *)c, ldc, M, N, K, ep, (int)wide_out);
    else hipLaunchKernelGGL((gemm_kernel<T, TA, TB, false>), grid, dim3(NT), 0, stream, (const T *)a, lda, (const T *)b, ldb, (T *)c, ldc, M, N, K, ep, (int)wide_out);
    return tokens_launch_status("linear");
}

// ---------------------------------------------------------------------------------------------- dz = dy act'(z), column sums
// A workgroup takes 64 columns x a run of rows: 16 column groups of 4 x 16 rows at a time.  Column sums are of the unrounded dz, one
// row of partial sums for each run, added up in a fixed order by the second kernel.
constexpr int DZ_COLS = 64;

template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const T *dy, int64_t lddy, const T *z, T *dz, float *part, int64_t M, int64_t N, int64_t run,
                                                 int act) {
    const int64_t n = (int64_t)blockIdx.x * DZ_COLS + (threadIdx.x & 15) * 4;
    const int64_t m1 = min(M, (int64_t)(blockIdx.y + 1) * run);
    const int left = n < N ? (int)min((int64_t)4, N - n) : 0;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t m = (int64_t)blockIdx.y * run + (threadIdx.x >> 4); m < m1; m += 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) {
                float g = (float)dy[m * lddy + n + i];
                if (act != BNDM_ACT_NONE) {
                    g *= act_slope(act, (float)z[m * N + n + i]);
                    dz[m * N + n + i] = (T)g;
                }
                sum[i] += g;
            }
    }
    if (!part) return;
    __shared__ float s[16][DZ_COLS];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[threadIdx.x >> 4][(threadIdx.x & 15) * 4 + i] = sum[i];
    __syncthreads();
    if (threadIdx.x < DZ_COLS) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += s[i][threadIdx.x];
        const int64_t col = (int64_t)blockIdx.x * DZ_COLS + threadIdx.x;
        if (col < N) part[(int64_t)blockIdx.y * N + col] = t;
    }
}

template <typename T> __global__ __launch_bounds__(256) void column_sums_kernel(const float *part, T *out, int64_t N, int runs) {
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float t = 0.f;
    for (int r = 0; r < runs; ++r) t += part[(int64_t)r * N + n];
    out[n] = (T)t;
}

// rows of a run: a workgroup's 256 threads take 16 rows at a time; at most 64 runs
int64_t rows_of_run(int64_t M) { return ceil_div64(ceil_div64(M, 64), 16) * 16; }
size_t dz_bytes(int64_t M, int64_t N, int act) { return act == BNDM_ACT_NONE ? 0 : (size_t)(((M * N * 2) + 255) / 256 * 256); }

template <typename T>
int backward(const void *dy, int64_t lddy, const void *z, const void *x, int64_t ldx, const void *w, void *dx, void *dw, void *dbias, int64_t M,
             int64_t N, int64_t K, int act, void *workspace, hipStream_t stream) {
    const void *dz = dy;
    int64_t lddz = lddy;
    if (act != BNDM_ACT_NONE || dbias) {
        float *part = dbias ? (float *)((char *)workspace + dz_bytes(M, N, act)) : nullptr;
        const int64_t run = rows_of_run(M);
        const int runs = (int)ceil_div64(M, run);
        hipLaunchKernelGGL((dz_kernel<T>), dim3((unsigned)ceil_div64(N, DZ_COLS), (unsigned)runs), dim3(256), 0, stream, (const T *)dy, lddy,
                           (const T *)z, (T *)workspace, part, M, N, run, act);
        if (int rc = tokens_launch_status("linear dz")) return rc;
        if (act != BNDM_ACT_NONE) dz = workspace, lddz = N;
        if (dbias) {
            hipLaunchKernelGGL((column_sums_kernel<T>), dim3((unsigned)ceil_div64(N, 256)), dim3(256), 0, stream, part, (T *)dbias, N, runs);
            if (int rc = tokens_launch_status("linear column sums")) return rc;
        }
    }
    const Epilogue none = {nullptr, nullptr, 0, nullptr, BNDM_ACT_NONE};
    if (dx)
        if (int rc = gemm<T, false, true>(dz, lddz, w, K, dx, K, M, K, N, none, stream)) return rc;
    if (dw)
        if (int rc = gemm<T, true, true>(dz, lddz, x, ldx, dw, K, N, K, M, none, stream)) return rc;
    return 0;
}

int check(const char *what, int64_t M, int64_t N, int64_t K, int act, int dtype) {
    TOKENS_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative size", what);
    TOKENS_REQUIRE(act == BNDM_ACT_NONE || act == BNDM_ACT_SILU || act == BNDM_ACT_GELU, "%s: activation %d", what, act);
    TOKENS_REQUIRE(dtype == BNDM_DTYPE_F16 || dtype == BNDM_DTYPE_BF16, "%s: dtype %d (f16 and bf16 only)", what, dtype);
    TOKENS_REQUIRE(M <= (1 << 23) && N <= (1 << 23) && K <= (1 << 23), "%s: sizes up to 2^23", what);
    return 0;
}

}  // namespace
}  // namespace bndm

using namespace bndm;

extern "C" int bndm_tokens_linear(const void *x, int64_t ldx, const void *w, const void *bias, const void *residual, int64_t ldr, void *y,
                                  void *z, int64_t M, int64_t N, int64_t K, int act, int dtype, void *stream) {
    if (int rc = check("bndm_tokens_linear", M, N, K, act, dtype)) return rc;
    if (M == 0 || N == 0) return 0;
    TOKENS_REQUIRE((x || K == 0) && (w || K == 0) && y, "bndm_tokens_linear: NULL tensor");
    TOKENS_REQUIRE(ldx >= 0 && ldx <= (1 << 23) && (!residual || ldr >= 0), "bndm_tokens_linear: row stride");
    const Epilogue ep = {bias, residual, ldr, z, act};
    if (dtype == BNDM_DTYPE_F16) return gemm<f16, false, false>(x, ldx, w, K, y, N, M, N, K, ep, (hipStream_t)stream);
    return gemm<bf16, false, false>(x, ldx, w, K, y, N, M, N, K, ep, (hipStream_t)stream);
}

extern "C" size_t bndm_tokens_linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int act, int want_dbias) {
    if (M <= 0 || N <= 0 || K < 0) return 0;
    return dz_bytes(M, N, act) + (want_dbias ? (size_t)ceil_div64(M, rows_of_run(M)) * N * 4 : 0);
}

extern "C" int bndm_tokens_linear_backward(const void *dy, int64_t lddy, const void *z, const void *x, int64_t ldx, const void *w, void *dx,
                                           void *dw, void *dbias, int64_t M, int64_t N, int64_t K, int act, int dtype, void *workspace,
                                           size_t workspace_bytes, void *stream) {
    if (int rc = check("bndm_tokens_linear_backward", M, N, K, act, dtype)) return rc;
    TOKENS_REQUIRE(M > 0 && N > 0 && K > 0, "bndm_tokens_linear_backward: empty layer");
    TOKENS_REQUIRE(dy && (act == BNDM_ACT_NONE || z) && (!dw || x) && (!dx || w), "bndm_tokens_linear_backward: NULL tensor");
    TOKENS_REQUIRE(ldx >= 0 && ldx <= (1 << 23) && lddy >= 0 && lddy <= (1 << 23), "bndm_tokens_linear_backward: row stride");
    const size_t need = bndm_tokens_linear_backward_workspace_bytes(M, N, K, act, dbias != nullptr);
    TOKENS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "bndm_tokens_linear_backward: workspace of %zu bytes, %zu needed",
                   workspace_bytes, need);
    if (dtype == BNDM_DTYPE_F16) return backward<f16>(dy, lddy, z, x, ldx, w, dx, dw, dbias, M, N, K, act, workspace, (hipStream_t)stream);
    return backward<bf16>(dy, lddy, z, x, ldx, w, dx, dw, dbias, M, N, K, act, workspace, (hipStream_t)stream);
}
