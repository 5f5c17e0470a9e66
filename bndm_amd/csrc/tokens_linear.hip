// Linear layer y = act(x W^T + b) + r and its gradients, on the matrix units.
//
//   forward   y[m][n]  = sum_k x[m][k] W[n][k]        both operands hold the summed index along their rows
//   dx        dx[m][k] = sum_n dz[m][n] W[n][k]       the second holds it across its rows
//   dW        dW[n][k] = sum_m dz[m][n] x[m][k]       both hold it across their rows
//
// One kernel takes all three: an operand whose rows run along the summed index is read from LDS as rows, one whose rows run across it
// by transposing LDS reads, so no operand is copied into another layout first.  Few rows go to a kernel of their own, which reads the
// weights straight into registers.
//
// Sums are 32 bits.  16 bits are, beside inputs and results: the kept z = x W^T + b, whose slope is taken (of 32 bits it would be twice the memory that a step
// keeps), and dz, because the matrix units multiply 16-bit operands.  Gradients are 1.4 times as far off as their own rounding leaves them.
#include "tokens_common.hpp"

namespace bndm {
namespace {

// ---------------------------------------------------------------------------------------------- activation
// Phi(-|z|) = exp(-z^2 / 2) t P(t) / 2 with t = 1 / (1 + 0.3 |z| / sqrt 2): P was fitted to exp(x^2) erfc(x).  With these coefficients it is off by
// 4.5e-8 of itself at most up to |z| = 14 (past which Phi(-|z|) is no normal number of 32 bits).  In 32 bits the whole is off by 5e-7 below
// |z| = 2, 1e-6 below 4 and 8e-6 near 13, where the rounding of the exponent is what counts; 1 + erf(z) has nothing left there.
struct Gauss { float below, density; };          // Phi(z), exp(-z^2 / 2) / sqrt(2 pi)
__device__ __forceinline__ Gauss gauss(float z) {
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.21213203435596426f * fabsf(z));
    const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
    float p = -0.12952277064323425f;
    p = __builtin_fmaf(p, t, 0.4855625629425049f);
    p = __builtin_fmaf(p, t, -0.5122767686843872f);
    p = __builtin_fmaf(p, t, 0.5477185845375061f);
    p = __builtin_fmaf(p, t, -0.09464973956346512f);
    p = __builtin_fmaf(p, t, 0.2149256467819214f);
    p = __builtin_fmaf(p, t, 0.14833927154541016f);
    p = __builtin_fmaf(p, t, 0.17071521282196045f);
    p = __builtin_fmaf(p, t, 0.1691880077123642f);
    const float tail = 0.5f * p * t * e;
    return {z < 0.f ? tail : 1.0f - tail, 0.39894228040143268f * e};
}
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z)); }

__device__ __forceinline__ float act_value(int act, float z) {
    if (act == BNDM_ACT_SILU) return z * logistic(z);
    if (act == BNDM_ACT_GELU) return z * gauss(z).below;
    return z;
}
// Past +-128 both slopes are 1 and 0 to 32 bits.  The kept z may be infinite there (f16 ends at 65504, its result from 32 bits need not be), where
// the formulas are 0 times infinity.
__device__ __forceinline__ float act_slope(int act, float z) {
    float slope;
    if (act == BNDM_ACT_SILU) {
        const float s = logistic(z);
        slope = s * (1.0f + z * (1.0f - s));
    } else {
        const Gauss g = gauss(z);
        slope = __builtin_fmaf(z, g.density, g.below);
    }
    return fabsf(z) > 128.0f ? (z > 0.f ? 1.0f : 0.0f) : slope;    // (a NaN stays one)
}

// ---------------------------------------------------------------------------------------------- what is done with a result
struct Epilogue {
    const void *bias;
    const void *residual;
    int64_t ldr;
    void *z;
    int act;
};

// 8 elements of a row, whatever its alignment; the first `left` of them where the row ends before
template <typename T> __device__ __forceinline__ s16x8 read8(const T *from, int left) {
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left >= 8) __builtin_memcpy(&v, from, 16);
    else
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) v[i] = reinterpret_cast<const short *>(from)[i];
    return v;
}
template <typename T> __device__ __forceinline__ void load8_of(float (&to)[8], const T *from, int left) {
    const s16x8 v = read8<T>(from, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) { const short s = v[i]; to[i] = widen<T>(s); }
}
template <typename T> __device__ __forceinline__ void store8_of(T *to, const float (&v)[8], int left) {
    const s16x8 p = pack8<T>(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
    if (left == 8) __builtin_memcpy(to, &p, 16);
    else
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) reinterpret_cast<short *>(to)[i] = p[i];
}

// What is added to 8 results of row m from column n on.  Both are read ahead of the results: read where they are added, 16384 x 1024 x
// 4096 with a residual took 209 us, this way 169 (150 without one).
template <typename T> __device__ __forceinline__ s16x8 bias8(const Epilogue &e, int64_t n, int64_t N) {
    return read8<T>((const T *)e.bias + n, e.bias && n < N ? (int)min((int64_t)8, N - n) : 0);
}
template <typename T> __device__ __forceinline__ s16x8 residual8(const Epilogue &e, int64_t m, int64_t n, int64_t M, int64_t N) {
    return read8<T>((const T *)e.residual + m * e.ldr + n, e.residual && m < M && n < N ? (int)min((int64_t)8, N - n) : 0);
}
// 8 consecutive results of row m from column n on (n < N)
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue &e, T *c, int64_t m, int64_t n, int64_t N, float (&v)[8], const s16x8 &bias, const s16x8 &residual) {
    const int left = (int)min((int64_t)8, N - n);
    float res[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const short b = bias[i], r = residual[i];
        v[i] += widen<T>(b);
        res[i] = widen<T>(r);
    }
    if (e.act == BNDM_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = act_value(BNDM_ACT_SILU, v[i]) + res[i];
    } else if (e.act == BNDM_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = act_value(BNDM_ACT_GELU, v[i]) + res[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[i] + res[i];
    }
    if (e.z) store8_of<T>((T *)e.z + m * N + n, v, left);
    store8_of<T>(c + m * N + n, y, left);
}

// ---------------------------------------------------------------------------------------------- the product
// C[m][n] = sum_k A(m, k) B(n, k).  TA false: A(m, k) = a[m * lda + k]; true: a[k * lda + m]; TB likewise.
// B's index runs down the registers of a result tile: a lane holds runs of 4 consecutive n of one row m.
// The tiles of a step of 32 of the summed index are copied into LDS three steps ahead of the products: with one step of 64 ahead, in the
// same 128 KB, 137 Gflop took 165 us, this way 131.
// 256 x 256 tiles are bound by the chip's power and the matrix units, and by a tile's end, which nothing overlaps: 16384 x 4096 x 1024 takes
// 132 us with W across (1040 Tflop/s; 128 at its least, the library's product 120), dW in four parts 132 and 14 to join them (940), 16384 x 1024 x 4096 with
// gelu and z kept 216 (640).  32768 x 512 x 512 with a residual takes 29 us, for 101 MB (3.5 TB/s).
constexpr int BK = 32;

// how operands come in: pieces of 16 bytes straight into LDS; through registers; element by element (rows of less than 8)
enum Loads { WIDE, ANY, NARROW };

struct Product {
    const void *a, *b;
    void *c;                       // [M][N]
    float *part;                   // splits > 1: [splits][M][N] sums of the parts of K
    int64_t lda, ldb, M, N, K;
    int64_t split_k;               // summed index of a part, a multiple of BK
    int tiles_m, tiles_n, tiles, splits;
};

// ROWS of one operand x 32 of the summed index in LDS, 16-byte chunks in swizzled places: rows along the summed index: [ROWS][4 chunks];
// across it: [32][ROWS / 8 chunks].  Copied by THREADS threads.
template <typename T, bool TR, int ROWS, int THREADS> struct Operand {
    static constexpr int C = TR ? ROWS / 8 : BK / 8;
    static constexpr int N = ROWS * (BK / 8) / THREADS;       // chunks of a thread
    static constexpr int STEP = THREADS / C;                  // rows between them
    static_assert(STEP % 16 == 0 || (TR && STEP == 8), "the swizzle's period is 16 rows, and 8 rows on it differs by 2");

    const char *base;              // where the tile of this step begins
    int64_t step_bytes;
    int row, c;                    // of the thread's first chunk
    int ld;
    int rows_in, inner_in;         // what is there from the tile of this step on: rows, elements of a row

    __device__ __forceinline__ static int place(int row) { return TR ? swizzle<16>(row) : swizzle<4>(row); }
    __device__ __forceinline__ void begin(const void *p, int64_t ld_, int64_t first_, int64_t extent, int64_t k0, int64_t k1, int tid) {
        ld = (int)ld_;
        base = (const char *)p + (TR ? k0 * ld_ + first_ : first_ * ld_ + k0) * 2;
        step_bytes = TR ? BK * ld_ * 2 : BK * 2;
        rows_in = (int)(TR ? k1 - k0 : extent - first_);
        inner_in = (int)(TR ? extent - first_ : k1 - k0);
        row = tid / C;
        c = (tid % C) ^ place(row);
    }
    __device__ __forceinline__ void next() {
        base += step_bytes;
        if constexpr (TR) rows_in -= BK;
        else inner_in -= BK;
    }
    __device__ __forceinline__ int chunk(int i) const { return STEP == 8 ? c ^ ((i & 1) << 1) : c; }
    __device__ __forceinline__ bool has(int i) const { return row + i * STEP < rows_in && chunk(i) * 8 < inner_in; }

    // every chunk is inside or outside as a whole: straight into LDS
    __device__ __forceinline__ void copy(char *lds, int w) const {
        const __amdgpu_buffer_rsrc_t rs = uniform_rsrc(base, kAnywhere);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t off = has(i) ? (uint32_t)((row + i * STEP) * ld + chunk(i) * 8) * 2u : kNowhere;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (i * THREADS + w * 64) * 16), 16, off, 0, 0, 0);
        }
    }
    // Any alignment, any size: through registers.  A chunk that the row's end cuts short is read as the row's last 8 elements and shifted
    // down when it is put away.  Past the end along the summed index are zeros; across it whatever is read there does, since its
    // results go nowhere: the last rows and chunks that are there.  So no load waits for another, and few tiles shift.
    struct Held { s16x8 v[N]; int left[N]; };
    __device__ __forceinline__ void load(Held &h) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row + i * STEP, at = chunk(i) * 8, left = inner_in - at;
            h.left[i] = TR ? (r >= rows_in ? 0 : left > 0 && left < 8 ? left : 8) : max(0, min(8, left));
            __builtin_memcpy(&h.v[i], (const short *)base + (int64_t)min(r, rows_in - 1) * ld + min(at, inner_in - 8), 16);
        }
    }
    // rows of less than 8 elements
    __device__ __forceinline__ void load_narrow(Held &h) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = chunk(i) * 8, left = left_of(i);
            const short *p = (const short *)base + (int64_t)(row + i * STEP) * ld + at;
            h.left[i] = 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) h.v[i][e] = e < left ? p[e] : (short)0;
        }
    }
    __device__ __forceinline__ int left_of(int i) const { return row + i * STEP < rows_in ? max(0, min(8, inner_in - chunk(i) * 8)) : 0; }
    __device__ __forceinline__ static void put(char *lds, const Held &h, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u64x2 v = __builtin_bit_cast(u64x2, h.v[i]);
            if (__any(h.left[i] != 8)) {
                const uint64_t lo = v.x, hi = v.y;
                const int by = 16 * (8 - h.left[i]);       // 0 .. 128
                v.x = by >= 64 ? hi >> (by & 63) : by ? (lo >> by) | (hi << (64 - by)) : lo;
                v.y = by >= 64 ? 0 : hi >> by;
                if (by == 128) v.x = 0;
            }
            *reinterpret_cast<u64x2 *>(lds + (i * THREADS + tid) * 16) = v;
        }
    }
};

// A lane's 8 values of row first + 32 block + l % 32 and k = 16 s + 8 (l / 32) .. + 7.
template <typename T, bool TR, int ROWS, int BLOCKS> struct Reader {
    static constexpr int BASES = TR ? 2 * BLOCKS : BK / 16;
    int at[BASES];

    __device__ __forceinline__ void begin(int first, int l) {
        const int h = l >> 5, i = l & 31;
        if constexpr (!TR) {
#pragma unroll
            for (int s = 0; s < BASES; ++s) at[s] = (first + i) * (BK * 2) + (((2 * s + h) ^ swizzle<4>(i)) << 4);
        } else {
            const int col = (l & 16) + 4 * (l & 3), k = 8 * h + ((l & 15) >> 2);
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    at[2 * b + u] = (k + 4 * u) * (ROWS * 2) + ((((first + 32 * b + col) >> 3) ^ swizzle<16>(k + 4 * u)) << 4) + (col & 4) * 2;
        }
    }
    __device__ __forceinline__ s16x8 read(const char *lds, int block, int s) const {
        if constexpr (!TR) return *reinterpret_cast<const s16x8 *>(lds + at[s] + block * 32 * BK * 2);
        else {
            const s16x4 lo = lds_read_tr(lds + at[2 * block] + s * 16 * ROWS * 2), hi = lds_read_tr(lds + at[2 * block + 1] + s * 16 * ROWS * 2);
            return join(lo, hi);
        }
    }
};

template <typename T, int FM, int FN, int A_BYTES, typename RA, typename RB>
__device__ __forceinline__ void products(const char *now, const RA &ra, const RB &rb, f32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
        s16x8 fa[FM], fb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = ra.read(now, i, kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = rb.read(now + A_BYTES, j, kk);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma32<T>(fb[j], fa[i], acc[i][j]);
    }
}

// One step: copies of a later one are sent off, then the products of this one.  The two pointers are __restrict__, and the function
// inlined, so that the compiler knows that the copies do not write what is read here: it would wait for them before the first read.
template <typename T, int FM, int FN, int A_BYTES, typename OA, typename OB, typename RA, typename RB>
__device__ __forceinline__ void step(char *__restrict__ ahead, const char *__restrict__ now, OA &oa, OB &ob, const RA &ra, const RB &rb,
                                     f32x16 (&acc)[FM][FN], int w) {
    oa.copy(ahead, w);
    ob.copy(ahead + A_BYTES, w);
    oa.next();
    ob.next();
    products<T, FM, FN, A_BYTES>(now, ra, rb, acc);
}

template <typename T, bool TA, bool TB, Loads LOADS, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void gemm_kernel(Product p, Epilogue ep) {
    constexpr int THREADS = 64 * (BM / WM) * (BN / WN), FM = WM / 32, FN = WN / 32;
    constexpr int A_BYTES = BM * BK * 2, STAGE = (BM + BN) * BK * 2;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Workgroups go to the 8 XCDs in turn: each gets a run of tiles, in groups of 8 tiles of rows, so that what runs at one time
    // behind one L2 shares its operands.
    const int per = (p.tiles * p.splits + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= p.tiles * p.splits) return;
    const int split = id / p.tiles, tile = id - split * p.tiles;
    const int group = tile / (8 * p.tiles_n), in_group = tile - group * 8 * p.tiles_n;
    const int high = min(8, p.tiles_m - group * 8);
    const int64_t m0 = (int64_t)(group * 8 + in_group % high) * BM, n0 = (int64_t)(in_group / high) * BN;
    const int wm = (w / (BN / WN)) * WM, wn = (w % (BN / WN)) * WN;

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int64_t k0 = split * p.split_k, k1 = min(p.K, k0 + p.split_k);
    const int steps = (int)((k1 - k0 + BK - 1) / BK);
    typedef Operand<T, TA, BM, THREADS> OA;
    typedef Operand<T, TB, BN, THREADS> OB;
    OA oa;
    OB ob;
    oa.begin(p.a, p.lda, m0, p.M, k0, k1, tid);
    ob.begin(p.b, p.ldb, n0, p.N, k0, k1, tid);
    Reader<T, TA, BM, FM> ra;
    Reader<T, TB, BN, FN> rb;
    ra.begin(wm, l);
    rb.begin(wn, l);
    if constexpr (LOADS == WIDE) {
        // (steps past the end are copied as well, as zeros without a read: the count of what is under way stays the same)
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            oa.copy(smem + s * STAGE, w);
            ob.copy(smem + s * STAGE + A_BYTES, w);
            oa.next();
            ob.next();
        }
        int slot = 0;
        for (int s = 0; s < steps; ++s) {
            // tile s is there (later ones may be under way), and tile s - 1 has been read by every wave
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * (OA::N + OB::N)) : "memory");
            const int to = slot + STAGES - 1;
            step<T, FM, FN, A_BYTES>(smem + (to >= STAGES ? to - STAGES : to) * STAGE, smem + slot * STAGE, oa, ob, ra, rb, acc, w);
            slot = slot + 1 == STAGES ? 0 : slot + 1;
        }
    } else {
        // AHEAD tiles in registers or on their way there while one is used.  (Tiles past the last are zeros and add nothing: no turn depends
        // on how many there are, or the compiler would wait for all loads wherever the paths meet.  Four ahead take no less time.)
        constexpr int AHEAD = 2;
        typename OA::Held va[AHEAD];
        typename OB::Held vb[AHEAD];
        auto fetch = [&](typename OA::Held &a, typename OB::Held &b) __attribute__((always_inline)) {
            if constexpr (LOADS == NARROW) {
                oa.load_narrow(a);
                ob.load_narrow(b);
            } else {
                oa.load(a);
                ob.load(b);
            }
            oa.next();
            ob.next();
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) fetch(va[u], vb[u]);
        for (int s = 0; s < steps; s += AHEAD)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                char *now = smem + (u & 1) * STAGE;
                OA::put(now, va[u], tid);                  // (the tile before the last, which lay here, has been read: every wave is past the last barrier)
                OB::put(now + A_BYTES, vb[u], tid);
                fetch(va[u], vb[u]);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                products<T, FM, FN, A_BYTES>(now, ra, rb, acc);
            }
    }
    wait_lds_dma();                                        // no copy is under way any more
    __syncthreads();
    // Results go through LDS, 32 rows x WN columns of a wave at a time, so that eight lanes write 128 bytes of a row: written from where
    // the products leave them, 8 bytes here and there, 134 MB took 70 us (1.9 TB/s).
    static_assert(WN == 64 && 8 * 1024 * (THREADS / 64) <= STAGES * STAGE, "a wave's 8 KB");
    char *own = smem + w * 8192;
    const int64_t n = n0 + wn + 8 * (l & 7);
    if (p.part) ep.bias = ep.residual = nullptr;           // (the kernel that joins the parts adds them)
    const s16x8 bias = bias8<T>(ep, n, p.N);
    s16x8 residual[2][4];
    auto ahead = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) residual[i & 1][t] = residual8<T>(ep, m0 + wm + 32 * i + 8 * t + (l >> 3), n, p.M, p.N);
    };
    ahead(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        if (i + 1 < FM) ahead(i + 1);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 v = {acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
                const int row = l & 31, chunk = 8 * j + (r >> 1) + (l >> 5);
                *reinterpret_cast<f32x4 *>(own + row * 256 + ((chunk ^ (row & 15)) << 4)) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int row = 8 * t + (l >> 3), chunk = 2 * (l & 7);
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(own + row * 256 + ((chunk ^ (row & 15)) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(own + row * 256 + (((chunk + 1) ^ (row & 15)) << 4));
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            const int64_t m = m0 + wm + 32 * i + row;
            if (m >= p.M || n >= p.N) continue;
            if (p.part) {
                float *to = p.part + ((int64_t)split * p.M + m) * p.N + n;
                if (n + 8 <= p.N) __builtin_memcpy(to, v, 32);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n + e < p.N) to[e] = v[e];
            } else finish8<T>(ep, (T *)p.c, m, n, p.N, v, bias, residual[i & 1][t]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// adds up the parts of K, in order
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Product p, Epilogue ep) {
    const int64_t chunks = (p.N + 7) / 8;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.M * chunks) return;
    const int64_t m = id / chunks, n = (id - m * chunks) * 8;
    const s16x8 bias = bias8<T>(ep, n, p.N), residual = residual8<T>(ep, m, n, p.M, p.N);
    float v[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        const float *from = p.part + ((int64_t)s * p.M + m) * p.N + n;
        if (n + 8 <= p.N) {
            float u[8];
            __builtin_memcpy(u, from, 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += u[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < p.N) v[e] += from[e];
        }
    }
    finish8<T>(ep, (T *)p.c, m, n, p.N, v, bias, residual);
}

// ---------------------------------------------------------------------------------------------- few rows
// A workgroup takes 16 columns and 16 MT rows; its 4 waves split the summed index, read both operands straight into registers
// (16 bytes of a row each, whatever its alignment) and join their sums in LDS.  What bounds it is the weights' way from memory and, below
// 10 MB of them, the time of two trips there: 4.0 us for 64 x 512 x 512, 4.8 us for 1 x 512 x 9984 (2.1 TB/s).
template <typename T, int MT> __global__ __launch_bounds__(256) void rows_kernel(Product p, Epilogue ep) {
    __shared__ float sums[4][16][16 * MT + 1];
    const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
    const int64_t n0 = (int64_t)(blockIdx.x / p.tiles_m) * 16, m0 = (int64_t)(blockIdx.x % p.tiles_m) * 16 * MT;
    const short *wp = (const short *)p.b + min(n0 + (l & 15), p.N - 1) * p.ldb;
    const short *xp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xp[t] = (const short *)p.a + min(m0 + 16 * t + (l & 15), p.M - 1) * p.lda;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto load = [&](const short *row, int64_t k) {
        s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (k + 8 <= p.K) __builtin_memcpy(&v, row + k, 16);
        else if (k < p.K)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < p.K) v[e] = row[k + e];
        return v;
    };
    const int64_t m = m0 + (tid >> 1), n = n0 + (tid & 1) * 8;   // of the results that this thread writes
    const s16x8 bias = bias8<T>(ep, n, p.N), residual = residual8<T>(ep, tid < 32 * MT ? m : p.M, n, p.M, p.N);
    // 128 of the summed index a turn, 4 steps for each wave at once
    for (int64_t k = (int64_t)w * 128; k < p.K; k += 512) {
        s16x8 wf[4], xf[4][MT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t at = k + 32 * s + 8 * (l >> 4);
            wf[s] = load(wp, at);
#pragma unroll
            for (int t = 0; t < MT; ++t) xf[s][t] = load(xp[t], at);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mfma16<T>(wf[s], xf[s][t], acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[w][4 * (l >> 4) + r][16 * t + (l & 15)] = acc[t][r];
    __syncthreads();
    if (tid >= 32 * MT || m >= p.M || n >= p.N) return;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int row = tid >> 1, col = (tid & 1) * 8 + e;
        v[e] = (sums[0][col][row] + sums[1][col][row]) + (sums[2][col][row] + sums[3][col][row]);
    }
    finish8<T>(ep, (T *)p.c, m, n, p.N, v, bias, residual);
}

// ---------------------------------------------------------------------------------------------- which kernel
struct Choice {
    int kind;                      // 0: few rows, 1: tiles of 128 x 128, 2: tiles of 256 x 256
    int splits, mt;
    int64_t split_k;
};

// The least of what the kernels take by this model, in us, fitted to 12 choices at each of 33 sizes from 1 x 4096 x 4096 to
// 16384 x 4096 x 1024 (rows x sum x columns), of which these are some, measured:
//                         rows kernel: 16 at a time,   32,    64;  128 x 128 tiles,  in 8 parts;  256 x 256 tiles
//   128 x 512 x 512                        3.6           4.1    5.0         9.8            10.3           19.1
//   512 x 512 x 512                        6.3           5.5    5.2         9.9            13.6           19.5
//   2048 x 512 x 512                      17.3          13.5   11.8        10.4              -            19.4
//   64 x 4096 x 4096                      31.8          25.9   22.5          -             16.3             -
//   128 x 4096 x 4096                     59.8          45.4   39.4        36.7            20.0           80.4
//   2048 x 2048 x 2048                      -           170    143         26.5              -            49.8
//   16384 x 4096 x 1024                     -             -      -         163               -            121
// A step of 64 along the sum takes a 128 x 128 tile 0.6 us alone on its CU and 1.15 with another one, a 256 x 256 tile 1.2 on a few
// CUs and 1.75 on all of them, half as much again through registers; the kernel for few rows reads 512 of the sum at a time.
Choice choose(int64_t M, int64_t N, int64_t K, bool rows_ok, bool wide) {
    Choice best = {1, 1, 1, K};
    double least = 1e300;
    for (int mt = 1; rows_ok && mt <= 4; mt *= 2) {
        const double blocks = (double)ceil_div64(M, 16 * mt) * (double)ceil_div64(N, 16);
        const double alone = mt == 1 ? 0.9 : mt == 2 ? 1.4 : 2.4, full = blocks * (mt == 1 ? 0.0036 : mt == 2 ? 0.0053 : 0.0091);
        const double us = 2.6 + (double)ceil_div64(K, 512) * (full > alone ? full : alone);
        if (us < least) least = us, best = {0, 1, mt, K};
    }
    const int64_t steps = ceil_div64(K, 64);
    for (int kind = 1; kind <= (wide ? 2 : 1); ++kind) {
        const int64_t t = kind == 2 ? 256 : 128, tiles = ceil_div64(M, t) * ceil_div64(N, t);
        for (int s = 1; s <= 16 && (s == 1 || (steps / s >= 4 && tiles * s <= 1024)); s *= 2) {
            const int64_t all = tiles * s, at_once = kind == 2 ? 256 : all <= 256 ? 256 : 512;
            const double step = kind == 2 ? 1.2 + 0.55 * (all < 256 ? all / 256.0 : 1.0) : (all <= 256 ? 0.6 : 1.15) * (wide ? 1.0 : 1.5);
            double us = (double)ceil_div64(all, at_once) * ((double)ceil_div64(steps, s) * step + (kind == 2 ? 9.0 : 4.5));
            if (s > 1) us += 3.0 + (double)M * (double)N * 8.0 * s / 5.0e6;
            if (us < least) least = us, best = {kind, s, 1, ceil_div64(steps, s) * 64};
        }
    }
    best.splits = best.kind == 0 || K == 0 ? 1 : (int)ceil_div64(K, best.split_k);
    return best;
}
size_t parts_bytes(const Choice &c, int64_t M, int64_t N) { return c.splits > 1 ? (size_t)c.splits * M * N * 4 : 0; }

template <typename T, bool TA, bool TB, Loads LOADS, int BM, int BN, int WM, int WN, int STAGES>
int launch_tiles(Product &p, const Epilogue &ep, hipStream_t stream) {
    constexpr int LDS = STAGES * (BM + BN) * BK * 2;
    const int64_t tiles = ceil_div64(p.M, BM) * ceil_div64(p.N, BN);
    TOKENS_REQUIRE(tiles * p.splits < (1 << 22), "linear: more tiles than a launch takes");
    p.tiles_m = (int)ceil_div64(p.M, BM), p.tiles_n = (int)ceil_div64(p.N, BN), p.tiles = (int)tiles;
    if constexpr (LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)gemm_kernel<T, TA, TB, LOADS, BM, BN, WM, WN, STAGES>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            tokens_error("linear: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
            return (int)e;
        }
    }
    hipLaunchKernelGGL((gemm_kernel<T, TA, TB, LOADS, BM, BN, WM, WN, STAGES>), dim3((unsigned)((tiles * p.splits + 7) / 8 * 8)),
                       dim3(64 * (BM / WM) * (BN / WN)), LDS, stream, p, ep);
    return tokens_launch_status("linear");
}

// `parts`: room for the parts of K (workspace), 16-byte aligned
template <typename T, bool TA, bool TB>
int gemm(const void *a, int64_t lda, const void *b, int64_t ldb, void *c, int64_t M, int64_t N, int64_t K, const Epilogue &ep, void *parts,
         hipStream_t stream) {
    // 16-byte loads: rows and the index along them in pieces of 8 elements (a piece is inside or outside as a whole)
    const bool wide_in = lda % 8 == 0 && ldb % 8 == 0 && (uint64_t)a % 16 == 0 && (uint64_t)b % 16 == 0 && (TA ? M : K) % 8 == 0 &&
                         (TB ? N : K) % 8 == 0;
    const Choice ch = choose(M, N, K, !TA && !TB, wide_in);
    Product p = {a, b, c, ch.splits > 1 ? (float *)parts : nullptr, lda, ldb, M, N, K, ch.split_k, 0, 0, 0, ch.splits};
    if constexpr (!TA && !TB)
        if (ch.kind == 0) {
            p.tiles_m = (int)ceil_div64(M, 16 * ch.mt);
            const int64_t blocks = ceil_div64(N, 16) * p.tiles_m;
            TOKENS_REQUIRE(blocks < (1 << 24), "linear: more tiles than a launch takes");
            if (ch.mt == 1) hipLaunchKernelGGL((rows_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, p, ep);
            else if (ch.mt == 2) hipLaunchKernelGGL((rows_kernel<T, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, p, ep);
            else hipLaunchKernelGGL((rows_kernel<T, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, p, ep);
            return tokens_launch_status("linear");
        }
    int rc;
    if ((TA ? M : K) < 8 || (TB ? N : K) < 8) rc = launch_tiles<T, TA, TB, NARROW, 128, 128, 64, 64, 2>(p, ep, stream);
    else if (!wide_in) rc = launch_tiles<T, TA, TB, ANY, 128, 128, 64, 64, 2>(p, ep, stream);
    else if (ch.kind == 2) rc = launch_tiles<T, TA, TB, WIDE, 256, 256, 128, 64, 4>(p, ep, stream);
    else rc = launch_tiles<T, TA, TB, WIDE, 128, 128, 64, 64, 4>(p, ep, stream);
    if (rc || ch.splits == 1) return rc;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)ceil_div64(M * ceil_div64(N, 8), 256)), dim3(256), 0, stream, p, ep);
    return tokens_launch_status("linear join");
}
// the largest that gemm() may take for either way of loading, which depends on addresses
size_t gemm_bytes(int64_t M, int64_t N, int64_t K, bool rows_ok) {
    const size_t a = parts_bytes(choose(M, N, K, rows_ok, true), M, N), b = parts_bytes(choose(M, N, K, rows_ok, false), M, N);
    return ((a > b ? a : b) + 255) / 256 * 256;
}

// ---------------------------------------------------------------------------------------------- dz = dy act'(z), column sums
// Bound by memory: 402 MB in 91 us (4.4 TB/s).
// A workgroup takes 256 columns x a run of rows, 8 columns a thread and 8 rows at a time.  Column sums are of the unrounded dz, one row
// of partial sums for each run, added up in a fixed order by the second kernel.
constexpr int DZ_COLS = 256;

template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const T *dy, int64_t lddy, const T *z, T *dz, float *part, int64_t M, int64_t N, int64_t run,
                                                 int act) {
    const int64_t n = (int64_t)blockIdx.x * DZ_COLS + (threadIdx.x & 31) * 8;
    const int64_t m1 = min(M, (int64_t)(blockIdx.y + 1) * run);
    const int left = n < N ? (int)min((int64_t)8, N - n) : 0;
    float sum[8] = {};
    if (left) {
#pragma unroll 2
        for (int64_t m = (int64_t)blockIdx.y * run + (threadIdx.x >> 5); m < m1; m += 8) {
            float g[8], zz[8] = {};
            load8_of<T>(g, dy + m * lddy + n, left);
            if (act != BNDM_ACT_NONE) load8_of<T>(zz, z + m * N + n, left);
            if (act == BNDM_ACT_SILU) {
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] *= act_slope(BNDM_ACT_SILU, zz[i]);
            } else if (act == BNDM_ACT_GELU) {
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] *= act_slope(BNDM_ACT_GELU, zz[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += g[i];
            if (act != BNDM_ACT_NONE) store8_of<T>(dz + m * N + n, g, left);
        }
    }
    if (!part) return;
    __shared__ float s[8][DZ_COLS];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[threadIdx.x >> 5][(threadIdx.x & 31) * 8 + i] = sum[i];
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += s[i][threadIdx.x];
    const int64_t col = (int64_t)blockIdx.x * DZ_COLS + threadIdx.x;
    if (col < N) part[(int64_t)blockIdx.y * N + col] = t;
}

// 32 columns a workgroup, 8 runs at a time
template <typename T> __global__ __launch_bounds__(256) void column_sums_kernel(const float *part, T *out, int64_t N, int runs) {
    __shared__ float s[8][32];
    const int64_t n = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    float t = 0.f;
    if (n < N)
#pragma unroll 4
        for (int r = threadIdx.x >> 5; r < runs; r += 8) t += part[(int64_t)r * N + n];
    s[threadIdx.x >> 5][threadIdx.x & 31] = t;
    __syncthreads();
    if (threadIdx.x < 32 && n < N) {
        t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += s[i][threadIdx.x];
        out[n] = (T)t;
    }
}

// rows of a run: 8 at least (a workgroup's rows at a time), about 2048 workgroups in all
int64_t rows_of_run(int64_t M, int64_t N) {
    const int64_t runs = ceil_div64(2048, ceil_div64(N, DZ_COLS));
    return ceil_div64(ceil_div64(M, runs), 8) * 8;
}
size_t dz_bytes(int64_t M, int64_t N, int act) { return act == BNDM_ACT_NONE ? 0 : (size_t)(((M * N * 2) + 255) / 256 * 256); }
size_t sums_bytes(int64_t M, int64_t N, bool want) { return want ? (size_t)((ceil_div64(M, rows_of_run(M, N)) * N * 4 + 255) / 256 * 256) : 0; }

template <typename T>
int backward(const void *dy, int64_t lddy, const void *z, const void *x, int64_t ldx, const void *w, void *dx, void *dw, void *dbias, int64_t M,
             int64_t N, int64_t K, int act, void *workspace, hipStream_t stream) {
    const void *dz = dy;
    int64_t lddz = lddy;
    char *parts = (char *)workspace + dz_bytes(M, N, act) + sums_bytes(M, N, dbias != nullptr);
    if (act != BNDM_ACT_NONE || dbias) {
        float *part = dbias ? (float *)((char *)workspace + dz_bytes(M, N, act)) : nullptr;
        const int64_t run = rows_of_run(M, N);
        const int runs = (int)ceil_div64(M, run);
        hipLaunchKernelGGL((dz_kernel<T>), dim3((unsigned)ceil_div64(N, DZ_COLS), (unsigned)runs), dim3(256), 0, stream, (const T *)dy, lddy,
                           (const T *)z, (T *)workspace, part, M, N, run, act);
        if (int rc = tokens_launch_status("linear dz")) return rc;
        if (act != BNDM_ACT_NONE) dz = workspace, lddz = N;
        if (dbias) {
            hipLaunchKernelGGL((column_sums_kernel<T>), dim3((unsigned)ceil_div64(N, 32)), dim3(256), 0, stream, part, (T *)dbias, N, runs);
            if (int rc = tokens_launch_status("linear column sums")) return rc;
        }
    }
    const Epilogue none = {nullptr, nullptr, 0, nullptr, BNDM_ACT_NONE};
    if (dx)
        if (int rc = gemm<T, false, true>(dz, lddz, w, K, dx, M, K, N, none, parts, stream)) return rc;
    if (dw)
        if (int rc = gemm<T, true, true>(dz, lddz, x, ldx, dw, N, K, M, none, parts, stream)) return rc;
    return 0;
}

int check(const char *what, int64_t M, int64_t N, int64_t K, int act, int dtype) {
    TOKENS_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative size", what);
    TOKENS_REQUIRE(act == BNDM_ACT_NONE || act == BNDM_ACT_SILU || act == BNDM_ACT_GELU, "%s: activation %d", what, act);
    TOKENS_REQUIRE(dtype == BNDM_DTYPE_F16 || dtype == BNDM_DTYPE_BF16, "%s: dtype %d (f16 and bf16 only)", what, dtype);
    TOKENS_REQUIRE(M <= (1 << 30) && N <= (1 << 22) && K <= (1 << 22), "%s: up to 2^30 rows, sizes up to 2^22", what);
    return 0;
}

}  // namespace
}  // namespace bndm

using namespace bndm;

extern "C" size_t bndm_tokens_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K < 0) return 0;
    return gemm_bytes(M, N, K, true);
}

extern "C" int bndm_tokens_linear(const void *x, int64_t ldx, const void *w, const void *bias, const void *residual, int64_t ldr, void *y,
                                  void *z, int64_t M, int64_t N, int64_t K, int act, int dtype, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    if (int rc = check("bndm_tokens_linear", M, N, K, act, dtype)) return rc;
    if (M == 0 || N == 0) return 0;
    TOKENS_REQUIRE((x || K == 0) && (w || K == 0) && y, "bndm_tokens_linear: NULL tensor");
    TOKENS_REQUIRE(ldx >= 0 && ldx <= (1 << 22) && (!residual || ldr >= 0), "bndm_tokens_linear: row stride");
    const size_t need = bndm_tokens_linear_workspace_bytes(M, N, K);
    TOKENS_REQUIRE(need == 0 || (workspace && (uint64_t)workspace % 16 == 0 && workspace_bytes >= need),
                   "bndm_tokens_linear: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const Epilogue ep = {bias, residual, ldr, z, act};
    if (dtype == BNDM_DTYPE_F16) return gemm<f16, false, false>(x, ldx, w, K, y, M, N, K, ep, workspace, (hipStream_t)stream);
    return gemm<bf16, false, false>(x, ldx, w, K, y, M, N, K, ep, workspace, (hipStream_t)stream);
}

extern "C" size_t bndm_tokens_linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int act, int want_dbias) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const size_t a = gemm_bytes(M, K, N, false), b = gemm_bytes(N, K, M, false);
    return dz_bytes(M, N, act) + sums_bytes(M, N, want_dbias) + (a > b ? a : b);
}

extern "C" int bndm_tokens_linear_backward(const void *dy, int64_t lddy, const void *z, const void *x, int64_t ldx, const void *w, void *dx,
                                           void *dw, void *dbias, int64_t M, int64_t N, int64_t K, int act, int dtype, void *workspace,
                                           size_t workspace_bytes, void *stream) {
    if (int rc = check("bndm_tokens_linear_backward", M, N, K, act, dtype)) return rc;
    TOKENS_REQUIRE(M > 0 && N > 0 && K > 0, "bndm_tokens_linear_backward: empty layer");
    TOKENS_REQUIRE(dy && (act == BNDM_ACT_NONE || z) && (!dw || x) && (!dx || w), "bndm_tokens_linear_backward: NULL tensor");
    TOKENS_REQUIRE(ldx >= 0 && ldx <= (1 << 22) && lddy >= 0 && lddy <= (1 << 22), "bndm_tokens_linear_backward: row stride");
    const size_t need = bndm_tokens_linear_backward_workspace_bytes(M, N, K, act, dbias != nullptr);
    TOKENS_REQUIRE(need == 0 || (workspace && (uint64_t)workspace % 16 == 0 && workspace_bytes >= need), "bndm_tokens_linear_backward: workspace of %zu bytes, %zu needed",
                   workspace_bytes, need);
    if (dtype == BNDM_DTYPE_F16) return backward<f16>(dy, lddy, z, x, ldx, w, dx, dw, dbias, M, N, K, act, workspace, (hipStream_t)stream);
    return backward<bf16>(dy, lddy, z, x, ldx, w, dx, dw, dbias, M, N, K, act, workspace, (hipStream_t)stream);
}
