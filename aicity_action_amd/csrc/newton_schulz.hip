// Newton-Schulz orthogonalisation of many matrices at once, and the Muon step around it.
//
//     X_0 = U / (|U|_F + eps)                                        (transposed where U is tall: m rows <= n columns)
//     A = X X^T,   B = b A + c A A,   X <- a X + B X                 (five times)
//
// pushes every singular value of X to about one.  A Muon step takes U from the momentum of a weight's gradient and the result as the
// weight's update.  All matrices of a call go through the same launches: one that reads the updates (and renews the momenta) and sums
// their squares, one that writes X_0, three products per iteration; a workgroup finds its matrix and tile in a table of kernel arguments.
//
// Arithmetic.  Products run on fp16 matrix cores with fp32 accumulators.  fp16 and not bf16: every operand is bounded (singular values
// of X stay below 1.3), so its range is enough with one power of two per operand, and it rounds eight times finer.  X itself is held as
// the sum of two fp16 values (22 bits): a gradient is dominated by a few directions, the rounding of whose entries lands in all the
// others, which five iterations amplify by up to a^5 = 485 -- with X in one fp16 value a rank-8 gradient over 1 % noise came out 4 %
// wrong, with two 0.04 % (384 x 1536, against 64 bits).  The products' own operands are the high halves: their rounding is that of one
// iteration and is not amplified (a full-rank gradient comes out 0.17 % wrong, which is their share).  SPLIT computes every product from
// both halves (high high + high low + low high, three times the matrix work): 5e-6 to 1e-5, for results wanted in single precision (4e-5 where one
// direction dominates: a rounding of X_0 is amplified by those 485, in single precision throughout as well).
//
// Bound by the matrix cores where matrices are large: 4096 x 4096 takes 1.72 ms = 800 TFLOP/s counting A and A A half (a large library product of
// this size: 1100), of which B X runs at 890; its LDS reads and LDS-DMA writes keep the LDS busy 1.5 times as long as the products the matrix
// cores.  By neither alone where they are many and shallow: the 34 M weights of the video model's blocks take 0.88 ms, of which a launch of B X moves
// 359 MB in 81 us (4.4 TB/s, counted) with the matrix cores busy for a quarter of it -- tiles of six steps mostly, whose first loads and way out
// do not overlap --, the squares and X_0 406 MB each in 74 and 72 us (5.5 and 5.6, what a copy reaches).
// By the latency of the chain of launches where they are few and small: 5 to 8 us each for three 1000 x 257, of which 2 are the launch's and the
// rest a first load, a few steps and the way out through LDS, one after the other.
#include "common.h"
#include <string.h>
#include <algorithm>
#include <type_traits>

typedef _Float16 h16;
typedef __attribute__((ext_vector_type(8))) _Float16 h16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 h16x4;
typedef __attribute__((address_space(3))) bf16x4 ns_lds_b4;

#define NS_MAX 72            // matrices per set of launches (kernel arguments hold their table)
#define NS_PARTS 256         // partial sums of squares per matrix
#define NS_SUMS 256          // partial tiles of 64 x 64 in the workspace
#define NS_BK 64             // depth of a K step; every matrix is padded with zeros to a multiple of it
// X, A and B are held times 2^12: their entries are at most their largest singular values (1.3, 1.6, 2.8 for the usual coefficients), so
// there is room to 16, and the low halves of entries down to 1e-4 are still normal fp16 numbers, which the matrix cores want
#define NS_S 4096.0f

// ---- what one set of launches works on --------------------------------------------------------------------------------------------
struct NsMat {               // reading side
    const void* u;           // update or gradient
    float* mom;              // momentum (Muon) or NULL
    int64_t rs, cs;          // element strides of u
    int32_t rows, cols;
    uint32_t off;            // start of the matrix' region in the workspace, in units of 64 fp16
    uint32_t first;          // first workgroup
};
struct NsLoadArgs {
    NsMat mat[NS_MAX];
    int n;
    uint32_t blocks;         // total workgroups
    h16* ws;
    double* parts;
    const float* norm_coef;  // {norm, factor} of all gradients, or NULL
    float mu;
    int nesterov;
    float eps;
};
struct NsGemmArgs {
    uint32_t first[NS_MAX];
    uint32_t off[NS_MAX];
    int32_t m[NS_MAX], n[NS_MAX];
    void* out[NS_MAX];       // last iteration: result or weight
    float scale[NS_MAX];     // last iteration: factor of the update (Muon)
    uint8_t tall[NS_MAX];
    int count;
    uint32_t blocks, run;    // tiles, and how many in a row go to one XCD
    uint32_t quarters;       // > 0: the tiles are the quarters of the tiles of 128 from quarters - 1 on (first counts tiles of 128)
    uint32_t cuts;           // NS_PART, NS_JOIN: pieces of every sum
    float* sums;             // ... and their partial tiles
    h16* ws;
    float a, b, c;
    int cur;                 // which of the two buffers holds the current X
    const float* norm_coef;
    const float* hyper;      // {lr, ...} in device memory or NULL
    float lr, wd;
};

__device__ __forceinline__ int ns_pad(int v) { return (v + 63) & ~63; }
// A matrix' region: X[0] high | X[1] high | X[0] low | A | B, and for SPLIT X[1] low | A low | B low.  X is an operand of the product that
// renews it, so it alternates between two buffers; its low half, which only the tile's own workgroup reads, stays in place without SPLIT.
struct NsRegion {
    h16* base;
    int64_t mn, mm;
    __device__ __forceinline__ NsRegion(h16* ws, uint32_t off, int m, int n)
        : base(ws + (int64_t)off * 64), mn((int64_t)ns_pad(m) * ns_pad(n)), mm((int64_t)ns_pad(m) * ns_pad(m)) {}
    __device__ __forceinline__ h16* x(int i) const { return base + i * mn; }
    __device__ __forceinline__ h16* xlo(int i) const { return i ? base + 3 * mn + 2 * mm : base + 2 * mn; }
    __device__ __forceinline__ h16* a() const { return base + 3 * mn; }
    __device__ __forceinline__ h16* b() const { return base + 3 * mn + mm; }
    __device__ __forceinline__ h16* alo() const { return base + 4 * mn + 2 * mm; }
    __device__ __forceinline__ h16* blo() const { return base + 4 * mn + 3 * mm; }
};
// Pins a value to fp32 before it is cut into a high and a low half.  Left to itself the compiler folds the product behind it and the
// conversion of one use into v_fma_mixlo_f16, which rounds once where the conversion of the other use rounds twice: about one value in
// 4000 then had a low half that did not belong to its high one.
template <typename T> __device__ __forceinline__ void ns_pin(T& v) { asm volatile("" : "+v"(v)); }

// the matrix a workgroup belongs to: the last one whose first workgroup is not behind it (one lane per entry of the table)
template <typename F>
__device__ __forceinline__ int ns_find(F first, int count, uint32_t blk) {
    const int lane = threadIdx.x & 63;
    const bool p0 = lane < count && first(lane) <= blk;
    const bool p1 = lane + 64 < count && first(lane + 64) <= blk;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(p0)) + __popcll(__ballot(p1)) - 1);
}

__device__ __forceinline__ bool ns_bad(const float* norm_coef) {       // (bit test: the build uses -fno-honor-nans)
    return norm_coef && (((__float_as_uint(norm_coef[0]) & 0x7f800000u) == 0x7f800000u) ||
                         ((__float_as_uint(norm_coef[1]) & 0x7f800000u) == 0x7f800000u));
}

// 2^12 / (norm + eps) as a mantissa and a power of two, applied one after the other: the factor itself leaves the range of fp32 for norms below
// 1e-35 and its precision for norms above 1e38.  An update of zeros stays one, however small eps is.
struct NsFactor {
    float mant;
    int exp;
    __device__ __forceinline__ float operator()(float v) const { return __builtin_ldexpf(v, exp) * mant; }
};
__device__ __forceinline__ NsFactor ns_factor(double squares, float eps) {
    const double f = squares == 0.0 ? 0.0 : (double)NS_S / (sqrt(squares) + (double)eps);
    return {(float)__builtin_amdgcn_frexp_mant(f), __builtin_amdgcn_frexp_exp(f)};
}

template <typename T> __device__ __forceinline__ float ns_ld(const T* p) { return ActIO<T>::load(p); }

// ---- 1. squares, and the momentum -------------------------------------------------------------------------------------------------
// M <- mu M + (1 - mu) c g;  u = Nesterov ? (1 - mu) c g + mu M : M.  The sum of squares is held in 64 bits (the squares of a gradient of
// 1e-20 are no fp32 numbers); every workgroup leaves one partial sum, which the next launch adds in order.
__device__ __forceinline__ float ns_update(const NsLoadArgs& a, float g, float m_new, float coef) {
    return a.nesterov ? (1.0f - a.mu) * (g * coef) + a.mu * m_new : m_new;
}

template <typename T>
__global__ __launch_bounds__(256) void ns_square_kernel(const NsLoadArgs a) {
    const int id = ns_find([&](int i) { return a.mat[i].first; }, a.n, blockIdx.x);
    const NsMat& t = a.mat[id];
    const uint32_t part = blockIdx.x - t.first;
    const uint32_t nparts = (id + 1 < a.n ? a.mat[id + 1].first : a.blocks) - t.first;
    const float coef = a.norm_coef ? a.norm_coef[1] : 1.0f;
    const bool bad = ns_bad(a.norm_coef);
    const T* u = static_cast<const T*>(t.u);
    double s = 0.0;
    const int64_t total = (int64_t)t.rows * t.cols;
    const bool flat_ok = t.cs == 1 && (t.rs == t.cols || t.rows == 1);
    if (flat_ok && sizeof(T) == 4 && ((reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(t.mom)) & 15) == 0) {
        const float4* u4 = reinterpret_cast<const float4*>(u);
        float4* m4 = reinterpret_cast<float4*>(t.mom);
        const int64_t n4 = total >> 2, step = (int64_t)nparts * 256;
        for (int64_t i0 = (int64_t)part * 256 + threadIdx.x; i0 < n4; i0 += 4 * step) {
            float4 g[4], m[4];                              // (four quads in flight; the last of them read again where there are fewer)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t i = i0 + q * step < n4 ? i0 + q * step : n4 - 1;
                g[q] = u4[i];
                if (t.mom) m[q] = m4[i];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (i0 + q * step >= n4) break;
                float4 v = g[q];
                if (t.mom) {
                    float4 p = m[q];
                    p.x = a.mu * p.x + (1.0f - a.mu) * (v.x * coef); p.y = a.mu * p.y + (1.0f - a.mu) * (v.y * coef);
                    p.z = a.mu * p.z + (1.0f - a.mu) * (v.z * coef); p.w = a.mu * p.w + (1.0f - a.mu) * (v.w * coef);
                    if (!bad) m4[i0 + q * step] = p;
                    v.x = ns_update(a, v.x, p.x, coef); v.y = ns_update(a, v.y, p.y, coef);
                    v.z = ns_update(a, v.z, p.z, coef); v.w = ns_update(a, v.w, p.w, coef);
                }
                s += ((double)v.x * v.x + (double)v.y * v.y) + ((double)v.z * v.z + (double)v.w * v.w);
            }
        }
        if (part == 0 && 4 * n4 + threadIdx.x < total) {     // at most three elements are left
            const int64_t i = 4 * n4 + threadIdx.x;
            float v = ns_ld(u + i);
            if (t.mom) {
                const float p = a.mu * t.mom[i] + (1.0f - a.mu) * (v * coef);
                if (!bad) t.mom[i] = p;
                v = ns_update(a, v, p, coef);
            }
            s += (double)v * (double)v;
        }
    } else {
        // neighbouring threads take neighbouring elements of u's own order, eight each in flight
        const bool by_col = t.cs == 1 || t.rs != 1;
        const int64_t inner = by_col ? t.cols : t.rows, step = (int64_t)nparts * 256;
        for (int64_t i0 = (int64_t)part * 256 + threadIdx.x; i0 < total; i0 += 8 * step) {
            float g[8], m[8];
            int64_t at[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int64_t i = i0 + q * step < total ? i0 + q * step : total - 1;
                if (flat_ok) {
                    at[q] = i;
                    g[q] = ns_ld(u + i);
                } else {
                    const int64_t o = i / inner, in = i - o * inner;
                    const int64_t r = by_col ? o : in, c = by_col ? in : o;
                    at[q] = r * t.cols + c;
                    g[q] = ns_ld(u + r * t.rs + c * t.cs);
                }
                if (t.mom) m[q] = t.mom[at[q]];
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (i0 + q * step >= total) break;
                float v = g[q];
                if (t.mom) {
                    const float p = a.mu * m[q] + (1.0f - a.mu) * (v * coef);
                    if (!bad) t.mom[at[q]] = p;
                    v = ns_update(a, v, p, coef);
                }
                s += (double)v * (double)v;
            }
        }
    }
    __shared__ double red[4];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.parts[(int64_t)id * NS_PARTS + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- 2. X_0 --------------------------------------------------------------------------------------------------------------------------
// One 64 x 64 tile of X per workgroup, through LDS (a tall update is transposed there), padding written as zeros.  The update is formed
// again from the gradient and the new momentum: the same bytes as writing it down and reading it back.
template <typename T>
__global__ __launch_bounds__(256) void ns_start_kernel(const NsLoadArgs a) {
    const int id = ns_find([&](int i) { return a.mat[i].first; }, a.n, blockIdx.x);
    const NsMat& t = a.mat[id];
    const bool tall = t.rows > t.cols;
    const int m = tall ? t.cols : t.rows, n = tall ? t.rows : t.cols;
    const int np = ns_pad(n);
    const uint32_t tile = blockIdx.x - t.first;
    const int per_row = np / 64;
    const int ti = tile / per_row, tj = tile - ti * per_row;       // tile row (of m), tile column (of n)
    const int tid = threadIdx.x;
    __shared__ float sh[64][65];                                    // [row of U][column of U] within the tile
    __shared__ double red[4];
    __shared__ NsFactor s_f;
    {
        const int64_t tiles = (int64_t)((t.rows + 63) / 64) * ((t.cols + 63) / 64);
        const int nparts = (int)(tiles < NS_PARTS ? tiles : NS_PARTS);
        double s = tid < nparts ? a.parts[(int64_t)id * NS_PARTS + tid] : 0.0;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
        if ((tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        if (tid == 0) s_f = ns_factor((red[0] + red[1]) + (red[2] + red[3]), a.eps);
    }
    const float coef = a.norm_coef ? a.norm_coef[1] : 1.0f;
    const T* u = static_cast<const T*>(t.u);
    const int r0 = (tall ? tj : ti) * 64, c0 = (tall ? ti : tj) * 64;   // the tile in U
    const bool by_col = t.cs == 1 || t.rs != 1;
    // every load is issued before the first is used, at clamped places; without Nesterov the update is the momentum itself
    const bool from_u = !t.mom || a.nesterov;
    const bool quads = sizeof(T) == 4 && t.cs == 1 && (t.rs & 3) == 0 && (t.cols & 3) == 0 &&
                       ((reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(t.mom)) & 15) == 0;
    if (quads) {
        float4 gv[4], mv[4];
        const int lc = (tid & 15) * 4, c = min(c0 + lc, t.cols - 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = min(r0 + (tid >> 4) + 16 * k, t.rows - 1);
            if (from_u) gv[k] = load4(u + (int64_t)r * t.rs + c);
            if (t.mom) mv[k] = load4(t.mom + (int64_t)r * t.cols + c);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int lr = (tid >> 4) + 16 * k;
            float v[4] = {gv[k].x, gv[k].y, gv[k].z, gv[k].w};
            if (t.mom) {
                const float mm[4] = {mv[k].x, mv[k].y, mv[k].z, mv[k].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = ns_update(a, v[j], mm[j], coef);
            }
            const bool in = r0 + lr < t.rows && c0 + lc < t.cols;
#pragma unroll
            for (int j = 0; j < 4; ++j) sh[lr][lc + j] = in ? v[j] : 0.f;
        }
    } else {
        float gv[16], mv[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int e = k * 256 + tid, lr = by_col ? e >> 6 : e & 63, lc = by_col ? e & 63 : e >> 6;
            const int r = min(r0 + lr, t.rows - 1), c = min(c0 + lc, t.cols - 1);
            if (from_u) gv[k] = ns_ld(u + (int64_t)r * t.rs + (int64_t)c * t.cs);
            if (t.mom) mv[k] = t.mom[(int64_t)r * t.cols + c];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int e = k * 256 + tid, lr = by_col ? e >> 6 : e & 63, lc = by_col ? e & 63 : e >> 6;
            const float v = t.mom ? ns_update(a, gv[k], mv[k], coef) : gv[k];
            sh[lr][lc] = r0 + lr < t.rows && c0 + lc < t.cols ? v : 0.f;
        }
    }
    __syncthreads();
    const NsFactor f = s_f;
    const NsRegion g(a.ws, t.off, m, n);
    // eight consecutive values of a row of X per thread
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int e = k * 256 + tid, row = e >> 3, ch = (e & 7) * 8;
        h16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = f(tall ? sh[ch + j][row] : sh[row][ch + j]);              // X[ti*64 + row][tj*64 + ch + j]
            ns_pin(v);
            hi[j] = (h16)v;
            lo[j] = (h16)(v - (float)hi[j]);
        }
        const int64_t ix = (int64_t)(ti * 64 + row) * np + tj * 64 + ch;
        *reinterpret_cast<h16x8*>(g.x(0) + ix) = hi;
        *reinterpret_cast<h16x8*>(g.xlo(0) + ix) = lo;
    }
}

// ---- 3. the products -----------------------------------------------------------------------------------------------------------------
// D[M][N] = sum_k P(k, M) Q[N][k]:  A = X X^T (P = Q = X) and A A (P = Q = A) with both operands contiguous in k, only tiles on and above
// the diagonal computed and each written twice;  X^T B^T = (B X)^T with P = X as it lies, k down its rows, read through the transposing LDS
// read, so that X is kept in one order.
// One workgroup = one T x T tile.  A group of four waves (2 x 2) takes K steps of 64 from a ring of D LDS stages of its own: the tile D - 1
// steps ahead is requested (LDS-DMA), then a step's fragments are read and its matrix instructions run while those ahead fly.  With G groups the
// steps are dealt in turn and the groups' sums added in order at the end.
// LDS: k-contiguous tiles have rows of 128 bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7): the 16 rows that a read serves together
// fall on 16 different slots of the 256-byte bank period.  X tiles as they lie have rows of 2 T bytes (a k each), 64-byte unit u of row r at
// u ^ (r & 3) (T = 128) or u ^ ((r >> 1) & 1) (T = 64): the four rows of a transposing read fall on different banks.
// The tile leaves through LDS in whole rows.  An accumulator register quad is four values along M, so [N][M] is the straight order:
// X itself, A, B, and the result of a wide matrix; the mirrored tiles of A and B and the result of a tall matrix are turned on the way.
// NS_PART computes one of the pieces of every sum of A = X X^T into the workspace, NS_JOIN adds them in order and goes on as NS_GRAM.
enum { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST16 = 3, NS_LAST32 = 4, NS_MUON = 5, NS_PART = 6, NS_JOIN = 7 };
__host__ __device__ constexpr bool ns_is_gram(int phase) { return phase == NS_GRAM || phase >= NS_PART; }
__host__ __device__ constexpr bool ns_is_last(int phase) { return phase >= NS_LAST16 && phase <= NS_MUON; }

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: a run of tiles, which share operand tiles, goes to one XCD.
__device__ __forceinline__ uint32_t ns_tile_of(uint32_t wg, uint32_t run) {
    const uint32_t xcd = wg & 7, slot = wg >> 3, r = slot / run;
    return (r * 8 + xcd) * run + (slot - r * run);
}

// 64 lanes x 16 bytes from base (wave-uniform) + offset to 1 KiB of LDS at dst (wave-uniform).  In asm because the compiler, which cannot tell
// these writes from the reads of the other stage, would wait for them in front of every read; the kernel waits itself (vmcnt) before its
// barriers.  (M0 cannot be named as overwritten; nothing else in the compiled kernels uses it, which a test reads from the object.)
__device__ __forceinline__ void ns_dma(const h16* base, uint32_t offset, const char* dst) {
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}

template <int T, int G, int D, int PHASE, bool SPLIT>
constexpr int ns_lds_bytes() {
    const int stages = G * D * (SPLIT ? 4 : 2) * T * 128;           // (the groups' sums lie within: behind the first group's stages)
    const int out = ns_is_last(PHASE) ? T * (T * 4 + 16) : 2 * T * (T * 2 + 16);
    return stages > out ? stages : out;
}

// waits until at most n stages of PER requests each are still on their way
template <int PER, int MOST>
__device__ __forceinline__ void ns_wait_stages(int n) {
    if constexpr (MOST == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (n >= MOST) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(PER * MOST) : "memory");
    else ns_wait_stages<PER, MOST - 1>(n);
}

template <int T, int G, int D, int PHASE, bool SPLIT>
__global__ __launch_bounds__(256 * G, G == 1 ? (SPLIT && T == 128 ? 1 : 2) : G) void ns_gemm_kernel(const NsGemmArgs a) {
    constexpr int F = T / 64;                      // 32 x 32 accumulators per wave and direction
    constexpr int PL = SPLIT ? 2 : 1;              // planes of an operand: high halves, low halves
    constexpr int STAGE = 2 * PL * T * 128;        // bytes of the P tiles + Q tiles of a step
    constexpr bool GRAM = ns_is_gram(PHASE), SYM = GRAM || PHASE == NS_POLY, LAST = ns_is_last(PHASE);
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const uint32_t blk = ns_tile_of(blockIdx.x, a.run);
    if (blk >= a.blocks) return;
    const bool quarter = T == 64 && a.quarters;
    const uint32_t unit = quarter ? a.quarters - 1 + blk / 4 : PHASE == NS_PART ? blk / a.cuts : blk;
    const int id = ns_find([&](int i) { return a.first[i]; }, a.count, unit);
    const int m = a.m[id], n = a.n[id], mp = ns_pad(m), np = ns_pad(n);
    const NsRegion g(a.ws, a.off[id], m, n);
    const uint32_t tile = unit - a.first[id];

    int tm, tn;
    if (SYM) {
        int J = (int)((sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while ((uint32_t)(J + 1) * (J + 2) / 2 <= tile) ++J;
        while ((uint32_t)J * (J + 1) / 2 > tile) --J;
        tn = J;
        tm = (int)(tile - (uint32_t)J * (J + 1) / 2);
    } else {
        // bands of eight tiles of B, through all of X: a run of tiles shares few of either
        const int side = quarter ? 128 : T;
        const uint32_t tiles_n = (mp + side - 1) / side, tiles_m = (np + side - 1) / side;
        const uint32_t band = tile / (8 * tiles_m), in_band = tile - band * 8 * tiles_m;
        const uint32_t width = min(8u, tiles_n - band * 8);
        tm = in_band / width;
        tn = band * 8 + (in_band - (uint32_t)tm * width);
    }
    const int lim_m = SYM ? mp : np, lim_n = mp;   // extents of the output
    if (quarter) {
        tm = 2 * tm + (int)(blk & 1);
        tn = 2 * tn + (int)(blk >> 1 & 1);
        if (tm * T >= lim_m || tn * T >= lim_n || (SYM && tm > tn)) return;
    }
    const int m0 = tm * T, n0 = tn * T;
    const int tid = threadIdx.x, grp = __builtin_amdgcn_readfirstlane(tid >> 8), wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
    const int lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wm = (wave & 1) * (T / 2), wn = (wave >> 1) * (T / 2);
    char* const lds = smem + grp * D * STAGE;

    // LDS-DMA: a wave instruction brings 1 KiB; waves 0 and 1 move P, waves 2 and 3 Q, T/16 pieces each.  Rows or columns past the padded
    // matrix are read again from its last ones; what comes of them is never stored
    constexpr int PW = T / 16;
    const bool is_q = wave >= 2;
    const bool by_k = !SYM && !is_q;               // the tile of X as it lies
    const int ldk = GRAM || !SYM ? np : mp;      // row length of P
    const int ld_src = is_q && !SYM ? mp : ldk;
    uint32_t src_off[PW];                          // byte offset of this lane's 16 bytes from the operand's tile
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int piece = (wave & 1) * PW + i;
        if (by_k) {
            const int row = piece * (512 / T) + lane / (T / 8), slot = lane % (T / 8);
            const int ch = T == 128 ? slot ^ ((row & 3) << 2) : slot ^ (((row >> 1) & 1) << 2);
            const int col = min(m0 + ch * 8, np - 8);
            src_off[i] = 2u * (uint32_t)(row * ld_src + col);
        } else {
            const int row = piece * 8 + (lane >> 3), ch = (lane & 7) ^ ((row >> 1) & 7);
            src_off[i] = 2u * (uint32_t)(min((is_q ? n0 : m0) + row, mp - 1) * ld_src + ch * 8);
        }
    }
    const int64_t k_step = by_k ? (int64_t)NS_BK * ld_src : NS_BK;
    int steps = (GRAM ? np : mp) / NS_BK, first_step = 0;
    if (PHASE == NS_PART) {
        const int per = (steps + (int)a.cuts - 1) / (int)a.cuts;
        first_step = (int)(blk - unit * a.cuts) * per;
        steps = max(0, min(per, steps - first_step));
    }
    if (PHASE == NS_JOIN) steps = 0;
    const int rounds = (steps + G - 1) / G, mine = (steps - grp + G - 1) / G;      // group 0 takes one in every round
    const h16* const src_hi = GRAM ? g.x(a.cur) : PHASE == NS_POLY ? g.a() : is_q ? g.b() : g.x(a.cur);
    const h16* const src_lo = GRAM ? g.xlo(a.cur) : PHASE == NS_POLY ? g.alo() : is_q ? g.blo() : g.xlo(a.cur);
    // a tile on the diagonal: Q is P, and is not loaded (20 x 2500, a single tile: 143 -> 127 us; nothing to gain where there are many)
    const bool same = SYM && T == 64 && tm == tn;
    auto dma = [=](int kt, int stage) {
        if (same && is_q) return;
        char* dst = lds + stage * STAGE + (is_q ? PL * T * 128 : 0) + (wave & 1) * PW * 1024;
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) {
            const h16* base = (pl ? src_lo : src_hi) + (kt + first_step) * k_step;
#pragma unroll
            for (int i = 0; i < PW; ++i) ns_dma(base, src_off[i], dst + pl * T * 128 + 1024 * i);
        }
    };

    // What is added to the product -- a X or b A -- comes through LDS too, in whole rows: the tile's halves are requested behind the last
    // step's tile (with two stages the low half follows when the sum is done).  16-byte chunk c of row r lies at c ^ (r & 15) (T = 128) or
    // c ^ ((r >> 1) & 7) (T = 64)
    constexpr bool RES = !GRAM, RES_LO = RES && (PHASE != NS_POLY || SPLIT);
    const h16* const res = PHASE == NS_POLY ? g.a() : g.x(a.cur);
    const h16* const reslo = PHASE == NS_POLY ? g.alo() : g.xlo(SPLIT ? a.cur : 0);
    auto res_dma = [=](const h16* src, int stage) {
        constexpr int PIECES = T * T / 2048;       // of a wave
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int piece = wave * PIECES + i;
            const int row = piece * (512 / T) + lane / (T / 8), slot = lane % (T / 8);
            const int ch = T == 128 ? slot ^ (row & 15) : slot ^ ((row >> 1) & 7);
            const int at = min(n0 + row, lim_n - 1) * lim_m + min(m0 + ch * 8, lim_m - 8);
            ns_dma(src, 2u * (uint32_t)at, lds + stage * STAGE + 1024 * piece);
        }
    };
    // a group's s-th request: its s-th step's tile, or behind the last one the residual's high half and low half
    auto request = [=](int s, int slot) {
        if (s < mine) dma(grp + s * G, slot);
        else if (RES && grp == 0) {
            if (s == mine) res_dma(res, slot);
            else if (RES_LO && D > 2 && s == mine + 1) res_dma(reslo, slot);
        }
    };
#pragma unroll
    for (int s = 0; s < D - 1; ++s) request(s, s);

    // the last iteration's result: its rows and columns; a weight's tile is requested here, to fly under the whole sum
    constexpr int QUADS = T * T / 4 / (256 * G);
    const bool tall = LAST && a.tall[id];
    const int R = tall ? n : m, C = tall ? m : n, row0 = tall ? m0 : n0, col0 = tall ? n0 : m0;
    const bool quads = LAST && (C & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out[id]) & (PHASE == NS_LAST16 ? 7 : 15)) == 0;
    float4 w[PHASE == NS_MUON ? QUADS : 1];
    if (PHASE == NS_MUON && quads)
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
            const int k = tid + 256 * G * i, row = k / (T / 4), c4 = (k - row * (T / 4)) * 4;
            w[PHASE == NS_MUON ? i : 0] = load4(static_cast<const float*>(a.out[id]) + (int64_t)min(row0 + row, R - 1) * C + min(col0 + c4, C - 4));
        }

    auto res_read = [=](int stage, int i, int j, int e4) {
        const int M = wm + 32 * i + 8 * e4 + 4 * h, N = wn + 32 * j + r;
        const int ch = T == 128 ? (M >> 3) ^ (N & 15) : (M >> 3) ^ ((N >> 1) & 7);
        return *reinterpret_cast<const h16x4*>(lds + stage * STAGE + N * (2 * T) + ch * 16 + (M & 4) * 2);
    };
    f32x16 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    float* const piece = PHASE >= NS_PART ? a.sums + (int64_t)(PHASE == NS_PART ? blk : unit * a.cuts) * 4096 + wave * 1024 + lane : nullptr;
    if (PHASE == NS_JOIN)
#pragma unroll 4
        for (uint32_t c = 0; c < a.cuts; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[0][0][e] += piece[(int64_t)c * 4096 + e * 64];

    const int q4 = (lane & 15) >> 2;               // transposing read: this lane names four columns of row 8 h + q4 (+ 4)
    const int tr_row = 8 * h + q4, tr_col = (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
    for (int it = 0, slot = 0, free = D - 1; it < rounds; ++it) {
        ns_wait_stages<PW * PL, D - 2>(mine - 1 - it);
        __syncthreads();                            // the step's tile has landed; everyone has read the stage refilled below
        if (G > 1 && it >= mine) continue;
        request(it + D - 1, free);
        h16x8 fp[PL][F][4], fq[PL][F][4];
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) {
            const char* sp = lds + slot * STAGE + pl * T * 128;
            const char* sq = same ? sp : sp + PL * T * 128;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    const int rp = wm + 32 * i + r, rq = wn + 32 * i + r;
                    if (SYM) fp[pl][i][ks] = *reinterpret_cast<const h16x8*>(sp + rp * 128 + (((2 * ks + h) ^ ((rp >> 1) & 7)) * 16));
                    else {
                        const int unit = (wm >> 5) + i, uu = T == 128 ? unit ^ q4 : unit ^ (q4 >> 1);
                        const char* at = sp + (16 * ks + tr_row) * (2 * T) + uu * 64 + tr_col;
                        const h16x4 lo = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ns_lds_b4*)at));
                        const h16x4 hi = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ns_lds_b4*)(at + 4 * 2 * T)));
                        fp[pl][i][ks] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    }
                    fq[pl][i][ks] = *reinterpret_cast<const h16x8*>(sq + rq * 128 + (((2 * ks + h) ^ ((rq >> 1) & 7)) * 16));
                }
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) {
                    if (SPLIT) {        // low high and high low first: they are small
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[PL - 1][i][ks], fq[0][j][ks], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][i][ks], fq[PL - 1][j][ks], acc[i][j], 0, 0, 0);
                    }
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][i][ks], fq[0][j][ks], acc[i][j], 0, 0, 0);
                }
        free = slot;
        slot = slot + 1 == D ? 0 : slot + 1;
    }

    const int res_slot = rounds % D, reslo_slot = (rounds + 1) % D;
    float* const sums = reinterpret_cast<float*>(smem + D * STAGE);
    if (RES || G > 1) {
        __syncthreads();
        if (RES_LO && D == 2 && grp == 0) res_dma(reslo, reslo_slot);
        if (G > 1 && grp > 0)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sums[(((grp - 1) * 4 + wave) * F * F + i * F + j) * 1024 + e * 64 + lane] = acc[i][j][e];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    // ---- the new values, times 2^12 but for the last iteration's ---------------------------------------------------------------------------
    if (PHASE == NS_PART) {
        if (grp == 0)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = acc[0][0][e];
#pragma unroll
                for (int o = 0; o < G - 1; ++o) v += sums[(o * 4 + wave) * 1024 + e * 64 + lane];
                piece[e * 64] = v;
            }
        return;
    }
    const float f_acc = PHASE == NS_POLY ? a.c / NS_S : LAST ? 1.0f / (NS_S * NS_S) : 1.0f / NS_S;
    const float f_res = PHASE == NS_POLY ? a.b : LAST ? a.a / NS_S : a.a;
    if (grp == 0)
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) {
                if (G > 1)          // the groups' sums, in order
#pragma unroll
                    for (int o = 0; o < G - 1; ++o)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][j][e] += sums[((o * 4 + wave) * F * F + i * F + j) * 1024 + e * 64 + lane];
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    h16x4 hi, lo;
                    if (RES) hi = res_read(res_slot, i, j, e4);
                    if (RES_LO) lo = res_read(reslo_slot, i, j, e4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& v = reinterpret_cast<float*>(&acc[i][j])[4 * e4 + e];
                        v *= f_acc;
                        if (RES) v += f_res * (RES_LO ? (float)hi[e] + (float)lo[e] : (float)hi[e]);
                    }
                }
                ns_pin(acc[i][j]);
            }

    if (LAST) {       // the result's rows through LDS in single precision
        constexpr int ROWB = T * 4 + 16;
        if (PHASE == NS_MUON && ns_bad(a.norm_coef)) return;
        __syncthreads();
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        const int M = wm + 32 * i + 8 * e4 + 4 * h, N = wn + 32 * j + r;
                        if (tall)
#pragma unroll
                            for (int e = 0; e < 4; ++e) *reinterpret_cast<float*>(smem + (M + e) * ROWB + N * 4) = acc[i][j][4 * e4 + e];
                        else
                            *reinterpret_cast<float4*>(smem + N * ROWB + M * 4) =
                                make_float4(acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2], acc[i][j][4 * e4 + 3]);
                    }
        __syncthreads();
        const float lr = a.hyper ? a.hyper[0] : a.lr;
        const float keep = 1.0f - lr * a.wd, step = lr * a.scale[id];
        if (quads) {
#pragma unroll
            for (int i = 0; i < QUADS; ++i) {
                const int k = tid + 256 * G * i, row = k / (T / 4), c4 = (k - row * (T / 4)) * 4;
                if (row0 + row >= R || col0 + c4 >= C) continue;
                const float4 v = *reinterpret_cast<const float4*>(smem + row * ROWB + c4 * 4);
                const int64_t at = (int64_t)(row0 + row) * C + col0 + c4;
                if (PHASE == NS_LAST16) store4(static_cast<bf16_t*>(a.out[id]) + at, v);
                else if (PHASE == NS_LAST32) store4(static_cast<float*>(a.out[id]) + at, v);
                else {
                    const float4 x = w[PHASE == NS_MUON ? i : 0];
                    store4(static_cast<float*>(a.out[id]) + at,
                           make_float4(x.x * keep - step * v.x, x.y * keep - step * v.y, x.z * keep - step * v.z, x.w * keep - step * v.w));
                }
            }
        } else {
#pragma unroll 4
            for (int k = tid; k < T * T; k += 256 * G) {
                const int row = k / T, c = k - row * T;
                if (row0 + row >= R || col0 + c >= C) continue;
                const float v = *reinterpret_cast<const float*>(smem + row * ROWB + c * 4);
                const int64_t at = (int64_t)(row0 + row) * C + col0 + c;
                if (PHASE == NS_LAST16) static_cast<bf16_t*>(a.out[id])[at] = f32_to_bf16(v);
                else if (PHASE == NS_LAST32) static_cast<float*>(a.out[id])[at] = v;
                else {
                    float* p = static_cast<float*>(a.out[id]) + at;
                    *p = *p * keep - step * v;
                }
            }
        }
        return;
    }

    // ---- the tile through LDS: X's high and low half in one pass; A and B and their mirror image, high halves, then (SPLIT) low halves ---------
    constexpr int ROWB = T * 2 + 16;
    const bool mirror = SYM && tm != tn;
    char* const o1 = smem;
    char* const o2 = smem + T * ROWB;
#pragma unroll
    for (int pass = 0; pass < (SYM && SPLIT ? 2 : 1); ++pass) {
        h16* const d1 = PHASE == NS_STEP ? g.x(a.cur ^ 1) : GRAM ? (pass ? g.alo() : g.a()) : (pass ? g.blo() : g.b());
        h16* const d2 = PHASE == NS_STEP ? g.xlo(SPLIT ? a.cur ^ 1 : 0) : d1;
        __syncthreads();
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        const int M = wm + 32 * i + 8 * e4 + 4 * h, N = wn + 32 * j + r;
                        h16x4 hi, lo;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = acc[i][j][4 * e4 + e];
                            hi[e] = (h16)x;
                            lo[e] = (h16)(x - (float)hi[e]);
                        }
                        const h16x4 v = pass ? lo : hi;
                        *reinterpret_cast<h16x4*>(o1 + N * ROWB + M * 2) = v;
                        if (PHASE == NS_STEP) *reinterpret_cast<h16x4*>(o2 + N * ROWB + M * 2) = lo;
                        else if (mirror)
#pragma unroll
                            for (int e = 0; e < 4; ++e) *reinterpret_cast<h16*>(o2 + (M + e) * ROWB + N * 2) = v[e];
                    }
        __syncthreads();
        constexpr int CH = T / 8;                 // 16-byte chunks of a row
#pragma unroll 4
        for (int k = tid; k < T * CH; k += 256 * G) {
            const int row = k / CH, c8 = (k - row * CH) * 8;
            const bool straight = n0 + row < lim_n && m0 + c8 < lim_m;
            const int64_t at = (int64_t)(n0 + row) * lim_m + m0 + c8;
            if (straight) *reinterpret_cast<h16x8*>(d1 + at) = *reinterpret_cast<const h16x8*>(o1 + row * ROWB + c8 * 2);
            if (PHASE == NS_STEP) {
                if (straight) *reinterpret_cast<h16x8*>(d2 + at) = *reinterpret_cast<const h16x8*>(o2 + row * ROWB + c8 * 2);
            } else if (mirror && m0 + row < lim_m && n0 + c8 < lim_n)
                *reinterpret_cast<h16x8*>(d2 + (int64_t)(m0 + row) * lim_m + n0 + c8) = *reinterpret_cast<const h16x8*>(o2 + row * ROWB + c8 * 2);
        }
    }
}

// ---- 4. small matrices: everything in one workgroup -------------------------------------------------------------------------------------
// A matrix of at most 48 (SPLIT: 32) tiles of 32 x 32 that fits into the 160 KB of LDS with A (B takes its place) takes all iterations in one
// workgroup of sixteen waves, and a call of such matrices is one launch instead of seventeen of 4 to 7 us each (96 x 288 26 us, 128 x 384
// 56 / 70, in SPLIT 96 x 288 47 / 93; the four of the video model's first block with their momenta 37).  Its time is the latency of reads,
// products and barriers in a row: A from its upper tiles alone, a third fewer reads, took as long.
// X stays in the accumulators in single precision.  A lane holds a column of the array the matrix comes from, an accumulator quad four of
// its rows, so that global accesses are whole lines; LDS holds the fp16 copy (SPLIT: both halves) as Y[column][row], which is X where the matrix
// is tall and X^T where it is wide, and the products read it along its rows or, with the transposing read, down them as that asks.  Rows in
// LDS are 16 bytes longer than their values, so that the 16 rows a read serves together fall on different banks.
#define NS_SMALL_MAX 56
#define NS_SMALL_WAVES 16
#define NS_SMALL_LDS 163840
struct NsSmallMat {
    const void* u;
    float* mom;
    void* out;
    int64_t rs, cs;
    int32_t rows, cols;
    float scale;
    int32_t pad;
};
struct NsSmallArgs {
    NsSmallMat mat[NS_SMALL_MAX];
    const float* norm_coef;
    const float* hyper;
    float mu, eps, a, b, c, lr, wd;
    int nesterov, steps;
};
__host__ __device__ static inline int ns_pad32(int v) { return (v + 31) & ~31; }
static inline int64_t ns_small_bytes(int rows, int cols, bool split) {
    const int64_t mp = ns_pad32(rows < cols ? rows : cols), np = ns_pad32(rows < cols ? cols : rows);
    if (mp > 128 || mp * np > (split ? 32 : 48) * 1024) return -1;
    const int64_t y = rows > cols ? mp * (np * 2 + 16) : np * (mp * 2 + 16);
    const int64_t bytes = (split ? 2 : 1) * (y + mp * (mp * 2 + 16)) + 256;
    return bytes <= NS_SMALL_LDS ? bytes : -1;
}

// An array of R x C elements with element strides rs and cs as a buffer resource: reads past its end give zero, writes past it are dropped,
// so a tile's sixteen accesses need one address and no comparison of rows.  (The whole offset goes into the address register, which the
// hardware compares with the size; offsets of the padded extents fit 31 bits.)
template <typename T>
struct NsArray {
    __amdgpu_buffer_rsrc_t rsrc;
    int rs, cs;
    __device__ __forceinline__ NsArray(const void* p, int R, int C, int rs_, int cs_)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, ((R - 1) * rs_ + (C - 1) * cs_ + 1) * (int)sizeof(T), 0x27000)),
          rs(rs_ * (int)sizeof(T)), cs(cs_ * (int)sizeof(T)) {}
    __device__ __forceinline__ int at(int row, int col) const { return row * rs + col * cs; }
    __device__ __forceinline__ float load(int at, int row) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, at + row * rs, 0, 0));
        else return bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(rsrc, at + row * rs, 0, 0));
    }
    __device__ __forceinline__ void store(float v, int at, int row) const {
        if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rsrc, at + row * rs, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(v), rsrc, at + row * rs, 0, 0);
    }
};

template <int PHASE, typename T, int TPW, bool SPLIT, bool TALL>
__device__ __forceinline__ void ns_small_body(const NsSmallArgs& a, const NsSmallMat& t, char* smem) {
    constexpr int PL = SPLIT ? 2 : 1;
    typedef std::conditional_t<PHASE == NS_LAST16, bf16_t, float> out_t;
    const int R = t.rows, C = t.cols;
    const int rp = ns_pad32(R), cp = ns_pad32(C), mp = TALL ? cp : rp, np = TALL ? rp : cp;
    const int nb = mp / 32, row_tiles = rp / 32, tiles = row_tiles * (cp / 32);
    const int ldy = rp * 2 + 16, lda = mp * 2 + 16;             // bytes of a row of Y, and of A and B
    const int ypl = cp * ldy, apl = mp * lda;                   // bytes of a plane
    char* const sy = smem + 256;
    char* const sa = sy + PL * ypl;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane0 = threadIdx.x & 63;
    const float coef = a.norm_coef ? a.norm_coef[1] : 1.0f;
    const bool bad = ns_bad(a.norm_coef);
    // the wave's k-th tile: rows from 32 rt, columns from 32 ct of the array; element 4 e4 + e of lane (r, h): row 8 e4 + 4 h + e, column r
    auto tile_of = [=](int k, int& rt, int& ct) {
        const int tile = wave + NS_SMALL_WAVES * k;
        ct = tile / row_tiles;
        rt = tile - ct * row_tiles;
        return tile < tiles;
    };
    const int r0 = lane0 & 31, h0 = lane0 >> 5;
    auto read_all = [=](const auto& arr, f32x16 (&v)[TPW]) {
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
            int rt, ct;
            if (tile_of(k, rt, ct)) {
                const int at = arr.at(32 * rt + 4 * h0, 32 * ct + r0);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[k][e] = arr.load(at, 8 * (e >> 2) + (e & 3));
            }
        }
    };
    auto write_all = [=](const auto& arr, const f32x16 (&v)[TPW]) {
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
            int rt, ct;
            if (tile_of(k, rt, ct) && 32 * ct + r0 < C) {
                const int at = arr.at(32 * rt + 4 * h0, 32 * ct + r0);
#pragma unroll
                for (int e = 0; e < 16; ++e) arr.store(v[k][e], at, 8 * (e >> 2) + (e & 3));
            }
        }
    };
    f32x16 x[TPW];
#pragma unroll
    for (int k = 0; k < TPW; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[k][e] = 0.f;
    read_all(NsArray<T>(t.u, R, C, (int)t.rs, (int)t.cs), x);
    if (PHASE == NS_MUON) {
        const NsArray<float> arr(t.mom, R, C, C, 1);
        f32x16 mo[TPW];
#pragma unroll
        for (int k = 0; k < TPW; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) mo[k][e] = 0.f;
        read_all(arr, mo);
#pragma unroll
        for (int k = 0; k < TPW; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float g = x[k][e], v = a.mu * mo[k][e] + (1.0f - a.mu) * (g * coef);
                x[k][e] = a.nesterov ? (1.0f - a.mu) * (g * coef) + a.mu * v : v;
                mo[k][e] = v;
            }
        if (!bad) write_all(arr, mo);
    }
    double sq = 0.0;
#pragma unroll
    for (int k = 0; k < TPW; ++k) {
        int rt, ct;
        const bool ok = tile_of(k, rt, ct) && 32 * ct + r0 < C;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float v = ok && 32 * rt + 8 * (e >> 2) + 4 * h0 + (e & 3) < R ? x[k][e] : 0.f;
            x[k][e] = v;
            sq += (double)v * (double)v;
        }
    }
    {
        double* red = reinterpret_cast<double*>(smem);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sq += __shfl_xor(sq, off, 64);
        if (lane0 == 0) red[wave] = sq;
        __syncthreads();
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < NS_SMALL_WAVES; ++k) s += red[k];
        const NsFactor f = ns_factor(s, a.eps);
#pragma unroll
        for (int k = 0; k < TPW; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[k][e] = f(x[k][e]);
    }

    const std::true_type down{};
    const std::false_type along{};
    for (int it = 0; it < a.steps; ++it) {
        int lane = lane0;           // made anew every iteration: addresses are cheaper recomputed than kept in registers through all of them
        ns_pin(lane);
        const int r = lane & 31, h = lane >> 5, q4 = (lane & 15) >> 2, c16 = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        // four values along M of a tile into row N
        auto put = [=](char* dst, int ld, int plane, const float (&v)[4], int N, int M) {
            h16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float p = v[e];
                ns_pin(p);
                hi[e] = (h16)p;
                lo[e] = (h16)(p - (float)hi[e]);
            }
            *reinterpret_cast<h16x4*>(dst + N * ld + M * 2) = hi;
            if (SPLIT) *reinterpret_cast<h16x4*>(dst + plane + N * ld + M * 2) = lo;
        };
        // one 32 x 32 tile of sum_k P(k, M) Q(k, N): an operand's k runs along its rows, or down them (transposing read)
        auto start = [=](auto tr, const char* p, int ld, int at) {
            return decltype(tr)::value ? p + (8 * h + q4) * ld + (at + c16) * 2 : p + (at + r) * ld + 16 * h;
        };
        auto fetch = [=](auto tr, const char* p, int ld) {
            if (decltype(tr)::value) {
                const h16x4 lo = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ns_lds_b4*)p));
                const h16x4 hi = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ns_lds_b4*)(p + 4 * ld)));
                return (h16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            return *reinterpret_cast<const h16x8*>(p);
        };
        auto product = [=](auto trp, auto trq, const char* P, int ldp, int ppl, const char* Q, int ldq, int qpl, int M0, int N0, int K) {
            f32x16 acc;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0.f;
            const char* p0 = start(trp, P, ldp, M0);
            const char* q0 = start(trq, Q, ldq, N0);
            const int pk = decltype(trp)::value ? 16 * ldp : 32, qk = decltype(trq)::value ? 16 * ldq : 32;      // bytes of 16 steps of k
            auto chunk = [&](auto steps) {              // that many times 16 steps of k: all fragments requested, then the products
                constexpr int S = decltype(steps)::value;
                h16x8 fp[S][PL], fq[S][PL];
#pragma unroll
                for (int s = 0; s < S; ++s) {
#pragma unroll
                    for (int pl = 0; pl < PL; ++pl) {
                        fp[s][pl] = fetch(trp, p0 + pl * ppl, ldp);
                        fq[s][pl] = fetch(trq, q0 + pl * qpl, ldq);
                    }
                    p0 += pk;
                    q0 += qk;
                }
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    if (SPLIT) {
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[s][PL - 1], fq[s][0], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[s][0], fq[s][PL - 1], acc, 0, 0, 0);
                    }
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[s][0], fq[s][0], acc, 0, 0, 0);
                }
            };
            int k = 0;                                  // K is a multiple of 32
            for (; k + 64 <= K; k += 64) chunk(std::integral_constant<int, 4>{});
            if (k < K) chunk(std::integral_constant<int, 2>{});
            return acc;
        };
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
            int rt, ct;
            if (tile_of(k, rt, ct))
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4)
                    put(sy, ldy, ypl, {x[k][4 * e4], x[k][4 * e4 + 1], x[k][4 * e4 + 2], x[k][4 * e4 + 3]}, 32 * ct + r, 32 * rt + 8 * e4 + 4 * h);
        }
        __syncthreads();
        const int ti = wave / nb, tj = wave - ti * nb;          // the wave's tile of A and B
        if (wave < nb * nb) {
            const f32x16 acc = TALL ? product(along, along, sy, ldy, ypl, sy, ldy, ypl, 32 * ti, 32 * tj, np)
                                    : product(down, down, sy, ldy, ypl, sy, ldy, ypl, 32 * ti, 32 * tj, np);
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const float f = 1.0f / NS_S;
                put(sa, lda, apl, {f * acc[4 * e4], f * acc[4 * e4 + 1], f * acc[4 * e4 + 2], f * acc[4 * e4 + 3]}, 32 * tj + r, 32 * ti + 8 * e4 + 4 * h);
            }
        }
        __syncthreads();
        // (a wave without a tile sums nothing, so that all of them come to the one barrier; a sum that only some carry across it spills)
        const f32x16 square = product(along, along, sa, lda, apl, sa, lda, apl, 32 * ti, 32 * tj, wave < nb * nb ? mp : 0);
        __syncthreads();                                        // everyone has read A: each wave puts its tile of B in its tile's place
        if (wave < nb * nb) {
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int N = 32 * tj + r, M = 32 * ti + 8 * e4 + 4 * h;
                const h16x4 hi = *reinterpret_cast<const h16x4*>(sa + N * lda + M * 2);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)hi[e];
                if (SPLIT) {
                    const h16x4 lo = *reinterpret_cast<const h16x4*>(sa + apl + N * lda + M * 2);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += (float)lo[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = a.b * v[e] + a.c / NS_S * square[4 * e4 + e];
                put(sa, lda, apl, v, N, M);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
            int rt, ct;
            if (tile_of(k, rt, ct)) {
                const f32x16 acc = TALL ? product(down, along, sy, ldy, ypl, sa, lda, apl, 32 * rt, 32 * ct, mp)
                                        : product(along, along, sa, lda, apl, sy, ldy, ypl, 32 * rt, 32 * ct, mp);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[k][e] = a.a * x[k][e] + acc[e] * (1.0f / NS_S);
            }
        }
        __syncthreads();
    }

    if (PHASE == NS_MUON) {
        if (bad) return;
        const float lr = a.hyper ? a.hyper[0] : a.lr;
        const float keep = 1.0f - lr * a.wd, step = lr * t.scale;
        const NsArray<float> arr(t.out, R, C, C, 1);
        f32x16 w[TPW];
        read_all(arr, w);
#pragma unroll
        for (int k = 0; k < TPW; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[k][e] = w[k][e] * keep - step * (x[k][e] * (1.0f / NS_S));
        write_all(arr, x);
    } else {
#pragma unroll
        for (int k = 0; k < TPW; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[k][e] *= 1.0f / NS_S;
        write_all(NsArray<out_t>(t.out, R, C, C, 1), x);
    }
}

template <int PHASE, typename T, int TPW, bool SPLIT>
__global__ __launch_bounds__(64 * NS_SMALL_WAVES) void ns_small_kernel(const NsSmallArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const NsSmallMat t = a.mat[blockIdx.x];
    if (t.rows > t.cols) ns_small_body<PHASE, T, TPW, SPLIT, true>(a, t, smem);
    else ns_small_body<PHASE, T, TPW, SPLIT, false>(a, t, smem);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
static inline int64_t pad64(int64_t v) { return (v + 63) & ~(int64_t)63; }

static int64_t ns_region_units(int rows, int cols, int split) {       // units of 64 fp16
    const int64_t mp = pad64(rows < cols ? rows : cols), np = pad64(rows < cols ? cols : rows);
    return (split ? 4 * mp * np + 4 * mp * mp : 3 * mp * np + 2 * mp * mp) / 64;
}

static int ns_check(const mvit_ns_matrix* mats, int count) {
    if (!mats || count < 1) return MVIT_EINVAL;
    for (int i = 0; i < count; ++i) {
        const mvit_ns_matrix& t = mats[i];
        if (t.rows < 1 || t.cols < 1) return MVIT_EINVAL;
        if (pad64(t.rows) * pad64(t.cols) >= ((int64_t)1 << 31)) return MVIT_EUNSUPPORTED;      // 32-bit offsets within a matrix
        if (pad64(t.rows < t.cols ? t.rows : t.cols) > 46000) return MVIT_EUNSUPPORTED;
    }
    return MVIT_OK;
}

// What a matrix is computed with: matrices of at most 32 rows or columns always from pairs -- the rounding of their few entries of A and B does not
// average out (2 x 7: up to 1.4 % from single fp16 values), and their products are short.  A call that has such matrices beside larger ones and
// asks for fp16 products runs as two parts, one behind the other in the same workspace; any other call is one part.  Where the matrices of few rows
// need tiles, the second chain of launches costs more than pairs for larger matrices of up to 256 tiles (one per CU): then the call is one
// part from pairs.  A Muon step in us, as two parts / one from pairs: 20x2500 beside 200x333 199 / 140, beside 384x1152 215 / 157, 1000x1000 (256
// tiles) 245 / 246, 768x2304 (432) 265 / 227, 1500x1500 (576) 351 / 472; where they fit one workgroup the sides are about even (18x768, 1x300 and 77x1 beside
// 130x70, 513x129 and 200x333 138 / 127, 384x1152 151 / 153, 768x2304 199 / 225), and it stays two.
struct NsPart {
    const mvit_ns_matrix* mats;
    int count, only;             // only: -1 all matrices, 0 the larger ones, 1 those of few rows or columns
    bool split, small;           // small: every matrix of the part fits one workgroup
    static bool few(const mvit_ns_matrix& t) { return t.rows <= 32 || t.cols <= 32; }
    NsPart(const mvit_ns_matrix* m, int n, int which, bool pairs) : mats(m), count(n), only(which), split(pairs), small(true) {
        for (int i = 0; i < count; ++i) {
            if (!has(i)) continue;
            const mvit_ns_matrix& t = mats[i];
            const int64_t rs = t.row_stride, cs = t.col_stride, most = (int64_t)1 << 28;
            small = small && ns_small_bytes(t.rows, t.cols, split) > 0 && rs >= 0 && cs >= 0 && rs < most && cs < most &&
                    (ns_pad32(t.rows) - 1) * rs + (ns_pad32(t.cols) - 1) * cs < most;       // (31-bit byte offsets, padding included)
        }
    }
    bool has(int i) const { return only < 0 || only == (int)few(mats[i]); }
    // the next matrices of the part from `from` on, at most `most` of them; `from` moves behind the last one looked at
    int take(int& from, int most, int* which) const {
        int n = 0;
        for (; from < count && n < most; ++from)
            if (has(from)) which[n++] = from;
        return n;
    }
};
// calls f(part) for the call's parts in order, until one does not return MVIT_OK
template <typename F>
static int ns_parts(const mvit_ns_matrix* mats, int count, int asked, F f) {
    int few = 0;
    for (int i = 0; i < count; ++i) few += NsPart::few(mats[i]);
    if (asked || few == 0 || few == count) return f(NsPart(mats, count, -1, asked || few));
    const NsPart rows(mats, count, 1, true);
    int64_t tiles = 0;             // of the larger ones
    for (int i = 0; i < count; ++i)
        if (!rows.has(i)) tiles += pad64(mats[i].rows) / 64 * (pad64(mats[i].cols) / 64);
    if (!rows.small && tiles <= 256) return f(NsPart(mats, count, -1, true));
    const int rc = f(rows);
    return rc != MVIT_OK ? rc : f(NsPart(mats, count, 0, false));
}

extern "C" int mvit_ns_matrix_bytes(void) { return (int)sizeof(mvit_ns_matrix); }

// sets of at most NS_MAX matrices run one after the other in the same workspace
extern "C" int64_t mvit_newton_schulz_workspace_bytes(const mvit_ns_matrix* mats, int count, int split) {
    const int rc = ns_check(mats, count);
    if (rc != MVIT_OK) return rc;
    int64_t bytes = 0;
    const int rc2 = ns_parts(mats, count, split, [&](const NsPart& part) {
        if (part.small) return (int)MVIT_OK;
        int64_t most = 0;
        int which[NS_MAX], n;
        for (int from = 0; (n = part.take(from, NS_MAX, which)) > 0;) {
            int64_t units = 0;
            for (int i = 0; i < n; ++i) units += ns_region_units(mats[which[i]].rows, mats[which[i]].cols, part.split);
            most = std::max(most, units);
        }
        if (most > 0xffffffffLL) return (int)MVIT_EUNSUPPORTED;
        bytes = std::max(bytes, most * 128 + (int64_t)NS_MAX * NS_PARTS * 8 + (part.split ? NS_SUMS * 16384 : 0));
        return (int)MVIT_OK;
    });
    return rc2 != MVIT_OK ? rc2 : bytes;
}

// tiles of a launch at a tile side
static int64_t ns_tiles(const NsGemmArgs& g, int side, bool sym, uint32_t* first) {
    int64_t at = 0;
    for (int i = 0; i < g.count; ++i) {
        const int64_t mt = (pad64(g.m[i]) + side - 1) / side, nt = (pad64(g.n[i]) + side - 1) / side;
        if (first) first[i] = (uint32_t)at;
        at += sym ? mt * (mt + 1) / 2 : mt * nt;
    }
    return at;
}

template <int T, int G, int D, int PHASE, bool SPLIT>
static int ns_launch_as(NsGemmArgs& g, hipStream_t st, int64_t rest = 0) {
    constexpr bool SYM = ns_is_gram(PHASE) || PHASE == NS_POLY;
    constexpr int LDS = ns_lds_bytes<T, G, D, PHASE, SPLIT>();
    static DevFlags done;
    DevFlag flag = dev_flag(done);
    if (LDS > 65536 && !flag) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&ns_gemm_kernel<T, G, D, PHASE, SPLIT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                LDS) != hipSuccess)
            return MVIT_ELAUNCH;
        flag = true;
    }
    // rest: that many tiles of 128 at the end are left to a second launch, which takes their quarters (T = 64)
    const int64_t tiles = ns_tiles(g, rest ? 128 : T, SYM, g.first);
    if (tiles > 0x1fffff00) return MVIT_EUNSUPPORTED;
    g.quarters = T == 64 && rest ? (uint32_t)(tiles - rest) + 1 : 0;
    g.blocks = (uint32_t)(T == 64 && rest ? 4 * rest : tiles - rest) * (PHASE == NS_PART ? g.cuts : 1);
    // runs of about 32 tiles (16 and 64 measured the same), as many for every XCD
    const uint32_t rounds = (g.blocks + 255) / 256;
    g.run = (g.blocks + 8 * rounds - 1) / (8 * rounds);
    hipLaunchKernelGGL((ns_gemm_kernel<T, G, D, PHASE, SPLIT>), dim3(rounds * 8 * g.run), dim3(256 * G), LDS, st, g);
    return hipGetLastError() == hipSuccess ? MVIT_OK : MVIT_ELAUNCH;
}

// Tiles of 128 (one pair of stages: two workgroups per CU, SPLIT one) read each operand half as often as tiles of 64, but are a quarter
// as many and take longer each: they are taken from 512 tiles on, and where the sums are about equally long (one
// that outlives the others leaves the rest of the chip idle: the model's A = X X^T, 300 tiles, 54 us against 46) from 192 on, which is three for
// each four CUs; SPLIT: where every round of 256 is more than three quarters full.  All five iterations, in us, below 512 tiles with
// tiles of 64 / with this rule: 3000 x 4000 1185 / 1015, 2500 x 2500 724 / 606, 2048 x 3000 503 / 460, 3 x 600 x 2000 173 / 179; SPLIT 2500 x 2500
// 1550 / 1317, 3 x 1500 x 1500 995 / 877.
// Up to 64 tiles of 128 behind the last full round (528 = 512 + 16 in the A of 4096 x 4096) would keep the chip waiting for a whole sum: a second
// launch takes their quarters, on four times as many CUs and two groups of waves each.  4096 x 4096 1823 / 1697, 4000 x 4100 1989 / 1792; SPLIT
// 4817 / 4371.  (Sums of 16 steps or more; shorter ones are over before a launch is.)
// Tiles of 64: up to 512 of them two per CU, whose time is the latency of their steps, take five stages; from eight steps on and with at most one
// tile per CU two groups of waves share them.  (All five iterations of 768 x 2304: 168 us with two stages and four groups / 156; 384 x 1536 118 /
// 108; more tiles than that overlap each other: three stages measured as two.)  SPLIT, whose stages are twice as large, gains nothing from
// their number (A = X X^T of 768 x 2304: two groups with two stages 22 us, one with five 24).  There a sum of 16 steps or more on few tiles is
// cut, so that up to 256 CUs share it and a second launch adds the pieces: 768 x 2304 248 / 224, 200 x 2400 195 / 144, 100 x 2500 183 / 117,
// 20 x 2500 126 / 92.  (A step of fp16 operands takes a third of that: a launch more would cost what cutting saves.)
template <int PHASE, bool SPLIT>
static int ns_launch(NsGemmArgs& g, hipStream_t st) {
    constexpr bool SYM = PHASE == NS_GRAM || PHASE == NS_POLY;
    int longest = 0, longest_rest = 0;
    int64_t work = 0;                     // steps of all tiles of 128
    const int64_t t128 = ns_tiles(g, 128, SYM, nullptr), t64 = ns_tiles(g, 64, SYM, nullptr), slots = SPLIT ? 256 : 512;
    int64_t rest = t128 % slots, at = 0;
    for (int i = 0; i < g.count; ++i) {
        const int64_t mt = (pad64(g.m[i]) + 127) / 128, nt = (pad64(g.n[i]) + 127) / 128, tiles = SYM ? mt * (mt + 1) / 2 : mt * nt;
        const int steps = (int)(pad64(PHASE == NS_GRAM ? g.n[i] : g.m[i]) / NS_BK);
        at += tiles;
        work += tiles * steps;
        longest = std::max(longest, steps);
        if (at > t128 - rest) longest_rest = std::max(longest_rest, steps);
    }
    if (t128 < slots || rest > 64 || longest_rest < 16) rest = 0;
    const bool even = 4 * work >= 3 * t128 * longest;
    if constexpr (SPLIT) {
        if (t128 - rest > 192 * ((t128 - rest + 255) / 256) && (even || t128 >= 512)) {
            const int rc = ns_launch_as<128, 1, 2, PHASE, true>(g, st, rest);
            return rc != MVIT_OK || !rest ? rc : ns_launch_as<64, 2, 2, PHASE, true>(g, st, rest);
        }
        if constexpr (PHASE == NS_GRAM) {
            const int64_t cuts = std::min<int64_t>(std::min<int64_t>(8, NS_SUMS / t64), longest / 4);
            if (cuts >= 2 && longest >= 16) {
                g.cuts = (uint32_t)cuts;
                const int rc = ns_launch_as<64, 2, 2, NS_PART, true>(g, st);
                return rc != MVIT_OK ? rc : ns_launch_as<64, 1, 2, NS_JOIN, true>(g, st);
            }
        }
        if (longest >= 8 && t64 <= 256) return ns_launch_as<64, 2, 2, PHASE, true>(g, st);
    } else {
        if (t128 >= 512 || (t128 >= 192 && even)) {
            const int rc = ns_launch_as<128, 1, 2, PHASE, false>(g, st, rest);
            return rc != MVIT_OK || !rest ? rc : ns_launch_as<64, 2, 5, PHASE, false>(g, st, rest);
        }
        if (longest >= 8 && t64 <= 256) return ns_launch_as<64, 2, 5, PHASE, false>(g, st);
        if (t64 <= 512) return ns_launch_as<64, 1, 5, PHASE, false>(g, st);
    }
    return ns_launch_as<64, 1, 2, PHASE, SPLIT>(g, st);
}

template <bool SPLIT>
static int ns_iterate(NsGemmArgs& g, int steps, int last, hipStream_t st) {
    int rc;
    for (int it = 0; it < steps; ++it) {
        g.cur = it & 1;
        if ((rc = ns_launch<NS_GRAM, SPLIT>(g, st)) != MVIT_OK) return rc;
        if ((rc = ns_launch<NS_POLY, SPLIT>(g, st)) != MVIT_OK) return rc;
        if (it + 1 < steps) rc = ns_launch<NS_STEP, SPLIT>(g, st);
        else rc = last == NS_LAST16 ? ns_launch<NS_LAST16, SPLIT>(g, st)
                : last == NS_LAST32 ? ns_launch<NS_LAST32, SPLIT>(g, st) : ns_launch<NS_MUON, SPLIT>(g, st);
        if (rc != MVIT_OK) return rc;
    }
    return MVIT_OK;
}

struct NsCall {
    float a, b, c, eps;
    int steps, split, in_dtype, last;
    float mu, lr, wd;
    int nesterov;
    const float *norm_coef, *hyper;
};

template <int PHASE, typename T, int TPW, bool SPLIT>
static int ns_small_launch_as(const NsSmallArgs& g, int count, int lds, hipStream_t st) {
    static DevFlags done;
    DevFlag flag = dev_flag(done);
    if (!flag) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&ns_small_kernel<PHASE, T, TPW, SPLIT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                NS_SMALL_LDS) != hipSuccess)
            return MVIT_ELAUNCH;
        flag = true;
    }
    hipLaunchKernelGGL((ns_small_kernel<PHASE, T, TPW, SPLIT>), dim3(count), dim3(64 * NS_SMALL_WAVES), lds, st, g);
    return hipGetLastError() == hipSuccess ? MVIT_OK : MVIT_ELAUNCH;
}
template <int PHASE, typename T>
static int ns_small_launch(const NsSmallArgs& g, int count, int lds, int tiles, bool split, hipStream_t st) {
    if (split) return ns_small_launch_as<PHASE, T, 32 / NS_SMALL_WAVES, true>(g, count, lds, st);
    return tiles <= 32 ? ns_small_launch_as<PHASE, T, 32 / NS_SMALL_WAVES, false>(g, count, lds, st)
                       : ns_small_launch_as<PHASE, T, 48 / NS_SMALL_WAVES, false>(g, count, lds, st);
}

// All matrices of a part small: one launch (of up to 56) does everything.  A part with a larger one takes the launches of the larger one's anyway.
static int ns_run_small(const NsPart& part, const NsCall& k, hipStream_t st) {
    const bool muon = k.last == NS_MUON, split = part.split;
    int which[NS_SMALL_MAX], c;
    for (int from = 0; (c = part.take(from, NS_SMALL_MAX, which)) > 0;) {
        NsSmallArgs g;
        memset(&g, 0, sizeof g);
        int64_t lds = 0;
        int tiles = 0;
        for (int i = 0; i < c; ++i) {
            const mvit_ns_matrix& t = part.mats[which[i]];
            g.mat[i] = {t.u, muon ? t.momentum : nullptr, muon ? static_cast<void*>(t.w) : t.out, t.row_stride, t.col_stride, t.rows, t.cols, t.scale, 0};
            lds = std::max(lds, ns_small_bytes(t.rows, t.cols, split));
            tiles = std::max(tiles, ns_pad32(t.rows) / 32 * (ns_pad32(t.cols) / 32));
        }
        g.norm_coef = k.norm_coef; g.hyper = k.hyper;
        g.mu = k.mu; g.eps = k.eps; g.a = k.a; g.b = k.b; g.c = k.c; g.lr = k.lr; g.wd = k.wd;
        g.nesterov = k.nesterov; g.steps = k.steps;
        int rc;
        if (muon) rc = ns_small_launch<NS_MUON, float>(g, c, (int)lds, tiles, split, st);
        else if (k.in_dtype == MVIT_F32)
            rc = k.last == NS_LAST16 ? ns_small_launch<NS_LAST16, float>(g, c, (int)lds, tiles, split, st)
                                     : ns_small_launch<NS_LAST32, float>(g, c, (int)lds, tiles, split, st);
        else
            rc = k.last == NS_LAST16 ? ns_small_launch<NS_LAST16, bf16_t>(g, c, (int)lds, tiles, split, st)
                                     : ns_small_launch<NS_LAST32, bf16_t>(g, c, (int)lds, tiles, split, st);
        if (rc != MVIT_OK) return rc;
    }
    return MVIT_OK;
}

static int ns_run_tiled(const NsPart& part, const NsCall& k, void* workspace, hipStream_t st) {
    const bool muon = k.last == NS_MUON, split = part.split;
    const mvit_ns_matrix* const mats = part.mats;
    int order[NS_MAX], n;
    for (int from = 0; (n = part.take(from, NS_MAX, order)) > 0;) {
        NsLoadArgs l;
        NsGemmArgs g;
        memset(&l, 0, sizeof l);
        memset(&g, 0, sizeof g);
        l.n = g.count = n;
        l.parts = static_cast<double*>(workspace);
        g.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + (int64_t)NS_MAX * NS_PARTS * 8);
        l.ws = g.ws = reinterpret_cast<h16*>(reinterpret_cast<char*>(g.sums) + (split ? NS_SUMS * 16384 : 0));
        l.norm_coef = g.norm_coef = k.norm_coef;
        l.mu = k.mu; l.nesterov = k.nesterov; l.eps = k.eps;
        g.a = k.a; g.b = k.b; g.c = k.c; g.hyper = k.hyper; g.lr = k.lr; g.wd = k.wd;
        // the matrices with the longest sums first, so that no launch ends on them
        std::stable_sort(order, order + l.n, [&](int x, int y) { return (int64_t)mats[x].rows + mats[x].cols > (int64_t)mats[y].rows + mats[y].cols; });
        int64_t off = 0, blocks = 0;
        for (int i = 0; i < l.n; ++i) {
            const mvit_ns_matrix& t = mats[order[i]];
            const int64_t tiles = ((t.rows + 63) / 64) * (int64_t)((t.cols + 63) / 64);
            l.mat[i] = {t.u, muon ? t.momentum : nullptr, t.row_stride, t.col_stride, t.rows, t.cols, (uint32_t)off, (uint32_t)blocks};
            g.off[i] = (uint32_t)off;
            g.tall[i] = t.rows > t.cols;
            g.m[i] = t.rows < t.cols ? t.rows : t.cols;
            g.n[i] = t.rows < t.cols ? t.cols : t.rows;
            g.out[i] = muon ? static_cast<void*>(t.w) : t.out;
            g.scale[i] = t.scale;
            off += ns_region_units(t.rows, t.cols, split);
            blocks += tiles < NS_PARTS ? tiles : NS_PARTS;
        }
        l.blocks = (uint32_t)blocks;
        if (k.in_dtype == MVIT_F32) hipLaunchKernelGGL(ns_square_kernel<float>, dim3(l.blocks), dim3(256), 0, st, l);
        else hipLaunchKernelGGL(ns_square_kernel<bf16_t>, dim3(l.blocks), dim3(256), 0, st, l);
        MVIT_LAUNCH_CHECK();
        blocks = 0;
        for (int i = 0; i < l.n; ++i) {
            l.mat[i].first = (uint32_t)blocks;
            blocks += pad64(l.mat[i].rows) / 64 * (pad64(l.mat[i].cols) / 64);
        }
        if (blocks > 0x7fffffff) return MVIT_EUNSUPPORTED;
        l.blocks = (uint32_t)blocks;
        if (k.in_dtype == MVIT_F32) hipLaunchKernelGGL(ns_start_kernel<float>, dim3(l.blocks), dim3(256), 0, st, l);
        else hipLaunchKernelGGL(ns_start_kernel<bf16_t>, dim3(l.blocks), dim3(256), 0, st, l);
        MVIT_LAUNCH_CHECK();
        const int rc = split ? ns_iterate<true>(g, k.steps, k.last, st) : ns_iterate<false>(g, k.steps, k.last, st);
        if (rc != MVIT_OK) return rc;
    }
    return MVIT_OK;
}

static int ns_run(const mvit_ns_matrix* mats, int count, const NsCall& k, void* workspace, int64_t bytes, hipStream_t st) {
    const bool muon = k.last == NS_MUON;
    const int64_t need = mvit_newton_schulz_workspace_bytes(mats, count, k.split);
    if (need < 0) return (int)need;
    if (bytes < need || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 127) || k.steps < 1) return MVIT_EINVAL;
    for (int i = 0; i < count; ++i)
        if (!mats[i].u || (muon ? !mats[i].w || !mats[i].momentum : !mats[i].out)) return MVIT_EINVAL;
    return ns_parts(mats, count, k.split,
                    [&](const NsPart& part) { return part.small ? ns_run_small(part, k, st) : ns_run_tiled(part, k, workspace, st); });
}

extern "C" int mvit_newton_schulz(const mvit_ns_matrix* mats, int count, int in_dtype, int out_dtype, float a, float b, float c, int steps,
                                  float eps, int split, void* workspace, int64_t workspace_bytes, void* stream) {
    if ((in_dtype != MVIT_F32 && in_dtype != MVIT_BF16) || (out_dtype != MVIT_F32 && out_dtype != MVIT_BF16)) return MVIT_EDTYPE;
    const NsCall k = {a, b, c, eps, steps, split, in_dtype, out_dtype == MVIT_F32 ? NS_LAST32 : NS_LAST16, 0.f, 0.f, 0.f, 0, nullptr, nullptr};
    return ns_run(mats, count, k, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int mvit_muon_step(const mvit_ns_matrix* mats, int count, float lr, float weight_decay, float momentum, int nesterov, float a,
                              float b, float c, int steps, float eps, int split, const float* norm_coef, const float* hyper,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    const NsCall k = {a, b, c, eps, steps, split, MVIT_F32, NS_MUON, momentum, lr, weight_decay, nesterov, norm_coef, hyper};
    return ns_run(mats, count, k, workspace, workspace_bytes, as_stream(stream));
}
