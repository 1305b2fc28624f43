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
// both halves (high high + high low + low high, three times the matrix work): 1e-6, for results wanted in single precision.
#include "common.h"
#include <string.h>

typedef _Float16 h16;
typedef __attribute__((ext_vector_type(8))) _Float16 h16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 h16x4;
typedef __attribute__((address_space(1))) const void ns_gptr_t;
typedef __attribute__((address_space(3))) void ns_lptr_t;

#define NS_MAX 72            // matrices per set of launches (kernel arguments hold their table)
#define NS_PARTS 256         // partial sums of squares per matrix
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
    int lo_t;                // the last iteration comes next: it reads a tall matrix' low half in X^T's order
};
struct NsGemmArgs {
    uint32_t first[NS_MAX];
    uint32_t off[NS_MAX];
    int32_t m[NS_MAX], n[NS_MAX];
    void* out[NS_MAX];       // last iteration: result or weight
    float scale[NS_MAX];     // last iteration: factor of the update (Muon)
    uint8_t tall[NS_MAX];
    int count;
    uint32_t blocks;
    h16* ws;
    float a, b, c;
    int cur;                 // which of the two X^T buffers holds the current one
    int lo_t;                // as above, for the X that this launch writes
    const float* norm_coef;
    const float* hyper;      // {lr, ...} in device memory or NULL
    float lr, wd;
};

__device__ __forceinline__ int ns_pad(int v) { return (v + 63) & ~63; }
// A matrix' region: X high | X low | X^T[0] | X^T[1] | X^T[0] low | A | B, and for SPLIT X^T[1] low | A low | B low
struct NsRegion {
    h16* base;
    int64_t mn, mm;
    __device__ __forceinline__ NsRegion(h16* ws, uint32_t off, int m, int n)
        : base(ws + (int64_t)off * 64), mn((int64_t)ns_pad(m) * ns_pad(n)), mm((int64_t)ns_pad(m) * ns_pad(m)) {}
    __device__ __forceinline__ h16* x() const { return base; }
    __device__ __forceinline__ h16* xlo() const { return base + mn; }
    __device__ __forceinline__ h16* xt(int i) const { return base + (i ? 3 : 2) * mn; }
    __device__ __forceinline__ h16* a() const { return base + 5 * mn; }
    __device__ __forceinline__ h16* b() const { return base + 5 * mn + mm; }
    __device__ __forceinline__ h16* xtlo(int i) const { return i ? base + 5 * mn + 2 * mm : base + 4 * mn; }
    __device__ __forceinline__ h16* alo() const { return base + 6 * mn + 2 * mm; }
    __device__ __forceinline__ h16* blo() const { return base + 6 * mn + 3 * mm; }
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
    auto one = [&](float g, int64_t flat) {
        float v = g;
        if (t.mom) {
            const float m = a.mu * t.mom[flat] + (1.0f - a.mu) * (g * coef);
            if (!bad) t.mom[flat] = m;
            v = ns_update(a, g, m, coef);
        }
        s += (double)v * (double)v;
    };
    const int64_t total = (int64_t)t.rows * t.cols;
    const bool flat_ok = t.cs == 1 && (t.rs == t.cols || t.rows == 1);
    if (flat_ok && sizeof(T) == 4 && ((reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(t.mom)) & 15) == 0) {
        const float4* u4 = reinterpret_cast<const float4*>(u);
        float4* m4 = reinterpret_cast<float4*>(t.mom);
        const int64_t n4 = total >> 2;
        for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < n4; i += (int64_t)nparts * 256) {
            const float4 g = u4[i];
            float4 v = g;
            if (t.mom) {
                float4 m = m4[i];
                m.x = a.mu * m.x + (1.0f - a.mu) * (g.x * coef); m.y = a.mu * m.y + (1.0f - a.mu) * (g.y * coef);
                m.z = a.mu * m.z + (1.0f - a.mu) * (g.z * coef); m.w = a.mu * m.w + (1.0f - a.mu) * (g.w * coef);
                if (!bad) m4[i] = m;
                v.x = ns_update(a, g.x, m.x, coef); v.y = ns_update(a, g.y, m.y, coef);
                v.z = ns_update(a, g.z, m.z, coef); v.w = ns_update(a, g.w, m.w, coef);
            }
            s += ((double)v.x * v.x + (double)v.y * v.y) + ((double)v.z * v.z + (double)v.w * v.w);
        }
        if (part == 0)
            for (int64_t i = 4 * n4 + threadIdx.x; i < total; i += 256) one(ns_ld(u + i), i);
    } else {
        // neighbouring threads take neighbouring elements of u's own order
        const bool by_col = t.cs == 1 || t.rs != 1;
        const int64_t inner = by_col ? t.cols : t.rows;
        for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < total; i += (int64_t)nparts * 256) {
            const int64_t o = i / inner, in = i - o * inner;
            const int64_t r = by_col ? o : in, c = by_col ? in : o;
            one(ns_ld(u + r * t.rs + c * t.cs), r * t.cols + c);
        }
    }
    __shared__ double red[4];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.parts[(int64_t)id * NS_PARTS + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- 2. X_0 in both orders ----------------------------------------------------------------------------------------------------------
// One 64 x 64 tile of X per workgroup, through LDS, padding written as zeros.  The update is formed again from the gradient and the new
// momentum: the same bytes as writing it down and reading it back.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void ns_start_kernel(const NsLoadArgs a) {
    const int id = ns_find([&](int i) { return a.mat[i].first; }, a.n, blockIdx.x);
    const NsMat& t = a.mat[id];
    const bool tall = t.rows > t.cols;
    const int m = tall ? t.cols : t.rows, n = tall ? t.rows : t.cols;
    const int mp = ns_pad(m), np = ns_pad(n);
    const uint32_t tile = blockIdx.x - t.first;
    const int per_row = np / 64;
    const int ti = tile / per_row, tj = tile - ti * per_row;       // tile row (of m), tile column (of n)
    const int tid = threadIdx.x;
    __shared__ float sh[64][65];                                    // [row of U][column of U] within the tile
    __shared__ double red[4];
    __shared__ float s_inv;
    {
        const int64_t tiles = (int64_t)((t.rows + 63) / 64) * ((t.cols + 63) / 64);
        const int nparts = (int)(tiles < NS_PARTS ? tiles : NS_PARTS);
        double s = tid < nparts ? a.parts[(int64_t)id * NS_PARTS + tid] : 0.0;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
        if ((tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        if (tid == 0) s_inv = (float)(1.0 / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + (double)a.eps));
    }
    const float coef = a.norm_coef ? a.norm_coef[1] : 1.0f;
    const T* u = static_cast<const T*>(t.u);
    const int r0 = (tall ? tj : ti) * 64, c0 = (tall ? ti : tj) * 64;   // the tile in U
    const bool by_col = t.cs == 1 || t.rs != 1;
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
        const int e = k * 256 + tid;
        const int lr = by_col ? e >> 6 : e & 63, lc = by_col ? e & 63 : e >> 6;
        const int r = r0 + lr, c = c0 + lc;
        float v = 0.f;
        if (r < t.rows && c < t.cols) {
            v = ns_ld(u + (int64_t)r * t.rs + (int64_t)c * t.cs);
            if (t.mom) v = ns_update(a, v, t.mom[(int64_t)r * t.cols + c], coef);
        }
        sh[lr][lc] = v;
    }
    __syncthreads();
    const float f = s_inv * NS_S;
    const NsRegion g(a.ws, t.off, m, n);
    // eight consecutive values per thread: X rows (64 of n each), then X^T rows (64 of m each)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int e = k * 256 + tid, row = e >> 3, ch = (e & 7) * 8;
        h16x8 hi, lo, hit, lot;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float vx = (tall ? sh[ch + j][row] : sh[row][ch + j]) * f;          // X[ti*64 + row][tj*64 + ch + j]
            float vt = (tall ? sh[row][ch + j] : sh[ch + j][row]) * f;          // X^T[tj*64 + row][ti*64 + ch + j]
            ns_pin(vx);
            ns_pin(vt);
            hi[j] = (h16)vx; lo[j] = (h16)(vx - (float)hi[j]);
            hit[j] = (h16)vt; lot[j] = (h16)(vt - (float)hit[j]);
        }
        const int64_t ix = (int64_t)(ti * 64 + row) * np + tj * 64 + ch, it = (int64_t)(tj * 64 + row) * mp + ti * 64 + ch;
        *reinterpret_cast<h16x8*>(g.x() + ix) = hi;
        *reinterpret_cast<h16x8*>(g.xt(0) + it) = hit;
        if (SPLIT) {
            *reinterpret_cast<h16x8*>(g.xlo() + ix) = lo;
            *reinterpret_cast<h16x8*>(g.xtlo(0) + it) = lot;
        } else if (a.lo_t && tall) *reinterpret_cast<h16x8*>(g.xtlo(0) + it) = lot;
        else *reinterpret_cast<h16x8*>(g.xlo() + ix) = lo;
    }
}

// ---- 3. the products -----------------------------------------------------------------------------------------------------------------
// D[M][N] = sum_k P[M][k] Q[N][k] with both operands contiguous in k: A = X X^T (P = Q = X), A A (P = Q = A, symmetric), B X (P = X^T,
// Q = B) and, in the last iteration of a tall matrix, P = B, Q = X^T.  X is kept in both orders for this; A and B are symmetric: only
// tiles on and above the diagonal are computed, each written twice.
// One workgroup = one T x T tile, four waves in 2 x 2, K steps of 64 from two LDS stages: a step's fragments are read into registers, the
// next step's tile is requested (LDS-DMA), then the matrix instructions run while it flies.  LDS rows are 128 bytes; 16-byte chunk c of row
// r lies at c ^ ((r >> 1) & 7), so the 16 rows that a read serves together fall on 16 different slots of the 256-byte bank period.
// The tile leaves through LDS in whole rows, in the order [N][M] ("direct": an accumulator register quad is four values of one such row)
// and, where both orders are kept, [M][N].
enum { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST16 = 3, NS_LAST32 = 4, NS_MUON = 5 };

template <int T, int PHASE, bool SPLIT>
__global__ __launch_bounds__(256, 2) void ns_gemm_kernel(const NsGemmArgs a) {
    constexpr int F = T / 64;                      // 32 x 32 accumulators per wave and direction
    constexpr int STAGE = 2 * T * 128;             // bytes of P tile + Q tile
    constexpr int OROW = T * 2 + 16;               // bytes of an output row in LDS
    constexpr bool SYM = PHASE == NS_GRAM || PHASE == NS_POLY;
    constexpr bool LAST = PHASE >= NS_LAST16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const uint32_t blk = blockIdx.x;
    const int id = ns_find([&](int i) { return a.first[i]; }, a.count, blk);
    const int m = a.m[id], n = a.n[id], mp = ns_pad(m), np = ns_pad(n);
    const bool tall = a.tall[id];
    const NsRegion g(a.ws, a.off[id], m, n);
    const uint32_t tile = blk - a.first[id];

    // operands and tile
    const h16 *p, *q, *plo = nullptr, *qlo = nullptr;
    int ldk, rows_p, rows_q, tm, tn;
    if (SYM) {
        int J = (int)((sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while ((uint32_t)(J + 1) * (J + 2) / 2 <= tile) ++J;
        while ((uint32_t)J * (J + 1) / 2 > tile) --J;
        tn = J;
        tm = (int)(tile - (uint32_t)J * (J + 1) / 2);
        rows_p = rows_q = mp;
        if (PHASE == NS_GRAM) { p = q = g.x(); plo = qlo = g.xlo(); ldk = np; }
        else { p = q = g.a(); plo = qlo = g.alo(); ldk = mp; }
    } else {
        ldk = mp;
        const bool swap = LAST && tall;
        p = swap ? g.b() : g.xt(a.cur);
        q = swap ? g.xt(a.cur) : g.b();
        if (SPLIT) { plo = swap ? g.blo() : g.xtlo(a.cur); qlo = swap ? g.xtlo(a.cur) : g.blo(); }
        rows_p = swap ? mp : np;
        rows_q = swap ? np : mp;
        const int tiles_m = (rows_p + T - 1) / T;
        tn = tile / tiles_m;
        tm = tile - tn * tiles_m;
    }
    const int m0 = tm * T, n0 = tn * T;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int r = lane & 31, h = lane >> 5;
    const int wm = (wave & 1) * (T / 2), wn = (wave >> 1) * (T / 2);

    // LDS-DMA: a wave instruction brings 8 rows of 128 bytes; wave w moves T/16 of the T/4 pieces (the first half is P)
    constexpr int PW = T / 16;
    const bool is_q = wave >= 2;
    int src_off[PW];                               // element offset of this lane's 16 bytes from the operand's tile column
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int row = ((wave & 1) * PW + i) * 8 + (lane >> 3);
        const int slot = lane & 7, ch = slot ^ ((row >> 1) & 7);
        const int lim = is_q ? rows_q : rows_p;
        int grow = (is_q ? n0 : m0) + row;
        grow = grow < lim ? grow : lim - 1;        // rows past the padded matrix: read again, never stored
        src_off[i] = grow * ldk + ch * 8;
    }
    const int nk = ldk / NS_BK;
    const int steps = SPLIT ? 3 * nk : nk;
    const h16* const src_hi = is_q ? q : p;
    const h16* const src_lo = is_q ? qlo : plo;
    auto dma = [=](int kt, int stage) {
        const h16* base = src_hi;
        if (SPLIT) {        // high high, then high low, then low high
            const int seg = kt >= 2 * nk ? 2 : kt >= nk ? 1 : 0;
            kt -= seg * nk;
            if (seg == (is_q ? 1 : 2)) base = src_lo;
        }
        base += kt * NS_BK;
        char* dst = smem + stage * STAGE + (is_q ? T * 128 : 0) + (wave & 1) * PW * 1024;
#pragma unroll
        for (int i = 0; i < PW; ++i)
            __builtin_amdgcn_global_load_lds((ns_gptr_t*)(base + src_off[i]), (ns_lptr_t*)(dst + 1024 * i), 16, 0, 0);
    };

    f32x16 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    dma(0, 0);
    for (int kt = 0; kt < steps; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                            // the step's tile has landed; everyone has read the stage refilled below
        const char* sp = smem + (kt & 1) * STAGE;
        h16x8 fp[F][4], fq[F][4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < F; ++i) {
                const int rp = wm + 32 * i + r, rq = wn + 32 * i + r;
                fp[i][ks] = *reinterpret_cast<const h16x8*>(sp + rp * 128 + (((2 * ks + h) ^ ((rp >> 1) & 7)) * 16));
                fq[i][ks] = *reinterpret_cast<const h16x8*>(sp + T * 128 + rq * 128 + (((2 * ks + h) ^ ((rq >> 1) & 7)) * 16));
            }
        if (kt + 1 < steps) dma(kt + 1, (kt + 1) & 1);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[i][ks], fq[j][ks], acc[i][j], 0, 0, 0);
    }

    // ---- epilogue: the new values in the accumulators -------------------------------------------------------------------------------
    const int lim_m = SYM ? mp : rows_p, lim_n = SYM ? mp : rows_q;      // extent of the output, both directions
    const h16* res = PHASE == NS_POLY ? g.a() : (LAST && tall) ? g.xt(a.cur) : g.x();
    const h16* reslo = PHASE == NS_POLY ? g.alo() : (LAST && tall) ? g.xtlo(SPLIT ? a.cur : 0) : g.xlo();
    const int64_t ldr = SYM ? mp : rows_p;                                // a row of the output [N][M]
    const float f_acc = PHASE == NS_POLY ? a.c / NS_S : LAST ? 1.0f / (NS_S * NS_S) : 1.0f / NS_S;
    const float f_res = PHASE == NS_POLY ? a.b : LAST ? a.a / NS_S : a.a;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int M = m0 + wm + 32 * i + 8 * e4 + 4 * h, N = n0 + wn + 32 * j + r;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (PHASE != NS_GRAM && M < lim_m && N < lim_n) {
                    const h16x4 hi = *reinterpret_cast<const h16x4*>(res + N * ldr + M);
                    x = make_float4((float)hi[0], (float)hi[1], (float)hi[2], (float)hi[3]);
                    if (PHASE != NS_POLY || SPLIT) {
                        const h16x4 lo = *reinterpret_cast<const h16x4*>(reslo + N * ldr + M);
                        x.x += (float)lo[0]; x.y += (float)lo[1]; x.z += (float)lo[2]; x.w += (float)lo[3];
                    }
                }
                float* v = reinterpret_cast<float*>(&acc[i][j]) + 4 * e4;
                v[0] = f_res * x.x + f_acc * v[0]; v[1] = f_res * x.y + f_acc * v[1];
                v[2] = f_res * x.z + f_acc * v[2]; v[3] = f_res * x.w + f_acc * v[3];
            }

    if (LAST) {       // rows of the result: N = the result's row, M its column
        const int R = tall ? n : m, C = tall ? m : n;
        const bool bad = PHASE == NS_MUON && ns_bad(a.norm_coef);
        const float lr = a.hyper ? a.hyper[0] : a.lr;
        const float keep = 1.0f - lr * a.wd, step = lr * a.scale[id];
        if (bad) return;
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int M = m0 + wm + 32 * i + 8 * e4 + 4 * h, N = n0 + wn + 32 * j + r;
                    if (N >= R) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (M + e >= C) continue;
                        const int64_t at = (int64_t)N * C + M + e;
                        const float v = acc[i][j][4 * e4 + e];
                        if (PHASE == NS_LAST16) static_cast<bf16_t*>(a.out[id])[at] = f32_to_bf16(v);
                        else if (PHASE == NS_LAST32) static_cast<float*>(a.out[id])[at] = v;
                        else {
                            float* w = static_cast<float*>(a.out[id]) + at;
                            *w = *w * keep - step * v;
                        }
                    }
                }
        return;
    }

    // ---- the tile through LDS: [N][M] and [M][N], high halves, then low halves ------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) ns_pin(acc[i][j]);
    h16* dst_d = PHASE == NS_GRAM ? g.a() : PHASE == NS_POLY ? g.b() : g.x();                 // [N][M]
    h16* dst_t = PHASE == NS_GRAM ? g.a() : PHASE == NS_POLY ? g.b() : g.xt(a.cur ^ 1);     // [M][N]
    const bool write_t = !SYM || tm != tn;
    const int ld_t = SYM ? mp : rows_q;
    const bool lo_in_t = PHASE == NS_STEP && !SPLIT && a.lo_t && tall;
    char* od = smem;
    char* ot = smem + T * OROW;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 1) {
            if (SYM && !SPLIT) break;
            dst_d = PHASE == NS_GRAM ? g.alo() : PHASE == NS_POLY ? g.blo() : g.xlo();
            dst_t = PHASE == NS_GRAM ? g.alo() : PHASE == NS_POLY ? g.blo() : g.xtlo(SPLIT ? a.cur ^ 1 : 0);
        }
        const bool do_d = pass == 0 || !lo_in_t;
        const bool do_t = write_t && (pass == 0 || SPLIT || lo_in_t);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int M = wm + 32 * i + 8 * e4 + 4 * h, N = wn + 32 * j + r;
                    h16x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = acc[i][j][4 * e4 + e];
                        const h16 hi = (h16)x;
                        v[e] = pass == 0 ? hi : (h16)(x - (float)hi);
                    }
                    if (do_d) *reinterpret_cast<h16x4*>(od + N * OROW + M * 2) = v;
                    if (do_t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) *reinterpret_cast<h16*>(ot + (M + e) * OROW + N * 2) = v[e];
                }
        __syncthreads();
        constexpr int CH = T / 8;                 // 16-byte chunks of a row
#pragma unroll 4
        for (int k = tid; k < T * CH; k += 256) {
            const int row = k / CH, c8 = (k - row * CH) * 8;
            if (do_d && n0 + row < lim_n && m0 + c8 < lim_m)
                *reinterpret_cast<h16x8*>(dst_d + (int64_t)(n0 + row) * ldr + m0 + c8) = *reinterpret_cast<const h16x8*>(od + row * OROW + c8 * 2);
            if (do_t && m0 + row < lim_m && n0 + c8 < lim_n)
                *reinterpret_cast<h16x8*>(dst_t + (int64_t)(m0 + row) * ld_t + n0 + c8) = *reinterpret_cast<const h16x8*>(ot + row * OROW + c8 * 2);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
static inline int64_t pad64(int64_t v) { return (v + 63) & ~(int64_t)63; }

static int64_t ns_region_units(int rows, int cols, int split) {       // units of 64 fp16
    const int64_t mp = pad64(rows < cols ? rows : cols), np = pad64(rows < cols ? cols : rows);
    return (split ? 6 * mp * np + 4 * mp * mp : 5 * mp * np + 2 * mp * mp) / 64;
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

extern "C" int mvit_ns_matrix_bytes(void) { return (int)sizeof(mvit_ns_matrix); }

// sets of at most NS_MAX matrices run one after the other in the same workspace
extern "C" int64_t mvit_newton_schulz_workspace_bytes(const mvit_ns_matrix* mats, int count, int split) {
    const int rc = ns_check(mats, count);
    if (rc != MVIT_OK) return rc;
    int64_t most = 0;
    for (int s = 0; s < count; s += NS_MAX) {
        int64_t units = 0;
        for (int i = s; i < count && i < s + NS_MAX; ++i) units += ns_region_units(mats[i].rows, mats[i].cols, split);
        if (units > most) most = units;
    }
    if (most > 0xffffffffLL) return MVIT_EUNSUPPORTED;
    return most * 128 + (int64_t)NS_MAX * NS_PARTS * 8;
}

template <int T, int PHASE, bool SPLIT>
static int ns_launch(NsGemmArgs& g, hipStream_t st) {
    constexpr int LDS = 2 * 2 * T * 128 > 2 * T * (T * 2 + 16) ? 2 * 2 * T * 128 : 2 * T * (T * 2 + 16);
    static DevFlags done;
    auto* kern = &ns_gemm_kernel<T, PHASE, SPLIT>;
    DevFlag flag = dev_flag(done);
    if (LDS > 65536 && !flag) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
            return MVIT_ELAUNCH;
        flag = true;
    }
    uint64_t at = 0;
    for (int i = 0; i < g.count; ++i) {
        const int64_t mt = (pad64(g.m[i]) + T - 1) / T, nt = (pad64(g.n[i]) + T - 1) / T;
        g.first[i] = (uint32_t)at;
        at += PHASE == NS_GRAM || PHASE == NS_POLY ? mt * (mt + 1) / 2 : mt * nt;
    }
    if (at > 0x7fffffffu) return MVIT_EUNSUPPORTED;
    g.blocks = (uint32_t)at;
    hipLaunchKernelGGL((ns_gemm_kernel<T, PHASE, SPLIT>), dim3(g.blocks), dim3(256), LDS, st, g);
    return hipGetLastError() == hipSuccess ? MVIT_OK : MVIT_ELAUNCH;
}

template <int T, bool SPLIT>
static int ns_iterate(NsGemmArgs& g, int steps, int last, hipStream_t st) {
    int rc;
    for (int it = 0; it < steps; ++it) {
        g.cur = it & 1;
        g.lo_t = it + 2 == steps;                 // the X written now is read by the last iteration
        if ((rc = ns_launch<T, NS_GRAM, SPLIT>(g, st)) != MVIT_OK) return rc;
        if ((rc = ns_launch<T, NS_POLY, SPLIT>(g, st)) != MVIT_OK) return rc;
        if (it + 1 < steps) rc = ns_launch<T, NS_STEP, SPLIT>(g, st);
        else rc = last == NS_LAST16 ? ns_launch<T, NS_LAST16, SPLIT>(g, st)
                : last == NS_LAST32 ? ns_launch<T, NS_LAST32, SPLIT>(g, st) : ns_launch<T, NS_MUON, SPLIT>(g, st);
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

static int ns_run(const mvit_ns_matrix* mats, int count, const NsCall& k, void* workspace, int64_t bytes, hipStream_t st) {
    const bool muon = k.last == NS_MUON;
    const int64_t need = mvit_newton_schulz_workspace_bytes(mats, count, k.split);
    if (need < 0) return (int)need;
    if (!workspace || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 127) || k.steps < 1) return MVIT_EINVAL;
    for (int i = 0; i < count; ++i)
        if (!mats[i].u || (muon ? !mats[i].w || !mats[i].momentum : !mats[i].out)) return MVIT_EINVAL;
    for (int s = 0; s < count; s += NS_MAX) {
        NsLoadArgs l;
        NsGemmArgs g;
        memset(&l, 0, sizeof l);
        memset(&g, 0, sizeof g);
        l.n = g.count = count - s < NS_MAX ? count - s : NS_MAX;
        l.parts = static_cast<double*>(workspace);
        l.ws = g.ws = reinterpret_cast<h16*>(static_cast<char*>(workspace) + (int64_t)NS_MAX * NS_PARTS * 8);
        l.norm_coef = g.norm_coef = k.norm_coef;
        l.mu = k.mu; l.nesterov = k.nesterov; l.eps = k.eps;
        l.lo_t = k.steps == 1;
        g.a = k.a; g.b = k.b; g.c = k.c; g.hyper = k.hyper; g.lr = k.lr; g.wd = k.wd;
        int64_t off = 0, blocks = 0;
        for (int i = 0; i < l.n; ++i) {
            const mvit_ns_matrix& t = mats[s + i];
            const int64_t tiles = ((t.rows + 63) / 64) * (int64_t)((t.cols + 63) / 64);
            l.mat[i] = {t.u, muon ? t.momentum : nullptr, t.row_stride, t.col_stride, t.rows, t.cols, (uint32_t)off, (uint32_t)blocks};
            g.off[i] = (uint32_t)off;
            g.tall[i] = t.rows > t.cols;
            g.m[i] = t.rows < t.cols ? t.rows : t.cols;
            g.n[i] = t.rows < t.cols ? t.cols : t.rows;
            g.out[i] = muon ? static_cast<void*>(t.w) : t.out;
            g.scale[i] = t.scale;
            off += ns_region_units(t.rows, t.cols, k.split);
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
        if (k.in_dtype == MVIT_F32) {
            if (k.split) hipLaunchKernelGGL((ns_start_kernel<float, true>), dim3(l.blocks), dim3(256), 0, st, l);
            else hipLaunchKernelGGL((ns_start_kernel<float, false>), dim3(l.blocks), dim3(256), 0, st, l);
        } else {
            if (k.split) hipLaunchKernelGGL((ns_start_kernel<bf16_t, true>), dim3(l.blocks), dim3(256), 0, st, l);
            else hipLaunchKernelGGL((ns_start_kernel<bf16_t, false>), dim3(l.blocks), dim3(256), 0, st, l);
        }
        MVIT_LAUNCH_CHECK();
        // tiles of 128 once there are enough of them to fill 256 CUs twice, else tiles of 64
        int64_t big = 0;
        for (int i = 0; i < l.n; ++i) big += (pad64(g.m[i]) + 127) / 128 * ((pad64(g.n[i]) + 127) / 128);
        int rc;
        if (big >= 512) rc = k.split ? ns_iterate<128, true>(g, k.steps, k.last, st) : ns_iterate<128, false>(g, k.steps, k.last, st);
        else rc = k.split ? ns_iterate<64, true>(g, k.steps, k.last, st) : ns_iterate<64, false>(g, k.steps, k.last, st);
        if (rc != MVIT_OK) return rc;
    }
    return MVIT_OK;
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
