// Rotary positions with several axes (time, height, width): each head's channels are cut into one section per axis, a section's channels
// into pairs (a, b), and the pair i of axis A turns by the angle p_A * f_i where p_A is the token's place on that axis:
//     y_a = x_a cos - x_b sin,     y_b = x_a sin + x_b cos;
// the scores q . k of rotated queries and keys then depend on the differences of places alone.  The transposed map is the turn by the
// negative angle, so the backward pass is the same kernel with the sine's sign flipped.  Channels behind the sections pass through; with
// an addend the result is rot(x) + add, rounded once.
//
// Bound by HBM: 2 * itemsize bytes and six operations per channel.  The angle is not read from a table: the place times the frequency (in
// turns) is one product in 64 bits -- a place of a million turns the fastest pair 160,000 times, which 32 bits would round to a hundredth
// of a turn -- whose fraction goes on in 32 bits (off by at most 2^-26 of a turn).  Sine and cosine of an eighth of a turn either way are
// their Taylor polynomials (next terms: 1.8e-9 and 1e-10), the quarter turn is put back by a swap and two signs.  All of it is shared by
// the rows that a thread walks: the heads of a batch entry, or of all of them where their places are the same.  Measured: 313 MB (bf16, one
// head, 8 clips of 8 x 112 x 112 tokens and their pooled keys) 63 us = 5.0 TB/s, 96 MB (8 x 28 x 28, four heads) 18.6 us = 5.2 TB/s, 658 MB
// (fp16, listed places around a million) 129 us = 5.1 TB/s; a large copy reaches 5.3 TB/s.  A call's time on the host is 12 us.
#include "common.h"
#include <algorithm>

struct RotaryArgs {
    mvit_rotary_tensor t[2];
    uint32_t first_block_1;        // blocks of t[1] begin here
    uint32_t blocks_per_group[2];  // blocks that cover L tokens x tasks of one group of rows
    uint32_t groups[2];            // groups of rows per span
    int rows_per_thread[2];        // rows = (batch, head) pairs
    int span[2];                   // rows that share their places: heads of one batch entry, or all
    int dim, pairs, axes;          // channels, rotated pairs of a head
    int tasks;                     // threads per token: pair chunks, then chunks of the channels that pass through
    int sec[MVIT_ROTARY_AXES];     // channels of each section
    float sign;
    double turns[MVIT_ROTARY_PAIRS];
};

template <typename T, int V> struct RotVec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct RotVec<T, 1> { typedef T type; };

template <typename T, int V>
__device__ __forceinline__ void rot_load(const T* p, float (&f)[V]) {
    const typename RotVec<T, V>::type v = *reinterpret_cast<const typename RotVec<T, V>::type*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        T e;
        if constexpr (V == 1) e = v;
        else e = v[j];
        if constexpr (sizeof(T) == 2) f[j] = bf16_to_f32(e);
        else f[j] = e;
    }
}
template <typename T, int V>
__device__ __forceinline__ void rot_store(T* p, const float (&f)[V]) {
    typename RotVec<T, V>::type v;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        T e;
        if constexpr (sizeof(T) == 2) e = f32_to_bf16(f[j]);
        else e = f[j];
        if constexpr (V == 1) v = e;
        else v[j] = e;
    }
    *reinterpret_cast<typename RotVec<T, V>::type*>(p) = v;
}

// The two vectors of a thread.  Interleaved pairs are 2 V channels side by side, aligned to V of them: one access (a dword pair needs no
// more than dword alignment).
template <typename T, int V> struct RotPair { typedef T type __attribute__((ext_vector_type(2 * V), aligned(V * sizeof(T)))); };
template <typename T, int V, bool INTER>
__device__ __forceinline__ void rot_load_pair(const T* p, int ca, int cb, float (&u)[V], float (&w)[V]) {
    if (INTER) {
        const typename RotPair<T, V>::type v = *reinterpret_cast<const typename RotPair<T, V>::type*>(p + ca);
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) {
            float f;
            if constexpr (sizeof(T) == 2) f = bf16_to_f32(v[j]);
            else f = v[j];
            if (j < V) u[j % V] = f;
            else w[j % V] = f;
        }
    } else {
        rot_load<T, V>(p + ca, u);
        rot_load<T, V>(p + cb, w);
    }
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ void rot_store_pair(T* p, int ca, int cb, const float (&u)[V], const float (&w)[V]) {
    if (INTER) {
        typename RotPair<T, V>::type v;
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) {
            const float f = j < V ? u[j % V] : w[j % V];
            if constexpr (sizeof(T) == 2) v[j] = f32_to_bf16(f);
            else v[j] = f;
        }
        *reinterpret_cast<typename RotPair<T, V>::type*>(p + ca) = v;
    } else {
        rot_store<T, V>(p + ca, u);
        rot_store<T, V>(p + cb, w);
    }
}

// sine and cosine of r turns, |r| <= 1/2
__device__ __forceinline__ void rot_sincos(float r, float& sn, float& cs) {
    const float q = __builtin_rintf(4.0f * r);
    const float t = 6.283185307179586f * fmaf(-0.25f, q, r), t2 = t * t;
    const float s = t * fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int n = (int)q;
    const uint32_t ss = __float_as_uint(n & 1 ? c : s), cc = __float_as_uint(n & 1 ? s : c);
    sn = __uint_as_float(ss ^ ((uint32_t)(n & 2) << 30));
    cs = __uint_as_float(cc ^ ((uint32_t)((n + 1) & 2) << 30));
}

// A thread owns V pairs of one token (2 V channels: two vectors of V) in up to rows_per_thread rows.  INTER: the pairs are (2i, 2i + 1),
// else (i, i + s / 2) within a section of s.  V divides what the host checked: every vector is aligned and none crosses a section's half
// (interleaved: pairs of two sections may share a thread, each pair looks up its own axis).
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    const int which = blockIdx.x >= a.first_block_1 ? 1 : 0;
    const mvit_rotary_tensor& t = a.t[which];
    const uint32_t blk = blockIdx.x - (which ? a.first_block_1 : 0u);
    const uint32_t row = blk / a.blocks_per_group[which], in_row = blk - row * a.blocks_per_group[which];
    const uint32_t item = in_row * 256u + threadIdx.x;
    const uint32_t l = item / (uint32_t)a.tasks, task = item - l * (uint32_t)a.tasks;
    if ((int64_t)l >= t.L) return;
    const uint32_t sp = row / a.groups[which], grp = row - sp * a.groups[which];
    const int r0 = (int)sp * a.span[which] + (int)grp * a.rows_per_thread[which];
    const int r1 = min(r0 + a.rows_per_thread[which], ((int)sp + 1) * a.span[which]);
    const uint32_t b = (uint32_t)r0 / (uint32_t)t.H;     // (one batch entry per span, or places shared by all)
    const int h0 = r0 - (int)b * t.H;

    const T* const x0 = static_cast<const T*>(t.x) + (int64_t)l * t.xs[2];
    T* const y0 = static_cast<T*>(t.y) + (int64_t)l * t.ys[2];
    const T* const add0 = t.add ? static_cast<const T*>(t.add) + (int64_t)l * t.as[2] : nullptr;
    const int p0 = (int)task * V;           // first pair of this thread
    const int chunks = a.pairs / V;

    if ((int)task >= chunks) {              // channels that pass through
        const int c0 = 2 * a.pairs + ((int)task - chunks) * 2 * V;
        int64_t bi = b, h = h0;
        for (int row = r0; row < r1; ++row) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = c0 + half * V;
                if (c >= a.dim) break;
                float f[V];
                rot_load<T, V>(x0 + bi * t.xs[0] + h * t.xs[1] + c, f);
                if (add0) {
                    float g[V];
                    rot_load<T, V>(add0 + bi * t.as[0] + h * t.as[1] + c, g);
#pragma unroll
                    for (int j = 0; j < V; ++j) f[j] += g[j];
                }
                rot_store<T, V>(y0 + bi * t.ys[0] + h * t.ys[1] + c, f);
            }
            if (++h == t.H) { h = 0; ++bi; }
        }
        return;
    }

    // the place on every axis
    double place[MVIT_ROTARY_AXES];
    if (t.pos) {
        const int64_t at = (int64_t)b * t.ps[0] + (int64_t)l * t.ps[1];
#pragma unroll
        for (int n = 0; n < MVIT_ROTARY_AXES; ++n) {
            if (n >= a.axes) break;
            const int64_t i = at + n * t.ps[2];
            place[n] = t.pos_type == MVIT_POS_I32 ? (double)static_cast<const int32_t*>(t.pos)[i]
                     : t.pos_type == MVIT_POS_I64 ? (double)static_cast<const int64_t*>(t.pos)[i]
                                                  : (double)static_cast<const float*>(t.pos)[i];
        }
    } else {
        uint32_t rest = l;
#pragma unroll
        for (int n = MVIT_ROTARY_AXES - 1; n >= 0; --n) {
            if (n >= a.axes) continue;
            const uint32_t q = rest / (uint32_t)t.grid[n];
            place[n] = t.origin[n] + t.step[n] * (double)(rest - q * (uint32_t)t.grid[n]);
            rest = q;
        }
    }
    float cs[V], sn[V];
    int ca = 2 * p0, cb = 2 * p0 + V;       // channels of the thread's two vectors
    int axis = 0, first = 0;                // axis of the pair, first channel of its section
    double at = place[0];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int p = p0 + j;
        if (INTER || j == 0) {              // (half: no vector crosses a section)
#pragma unroll
            for (int n = 1; n < MVIT_ROTARY_AXES; ++n)
                if (axis == n - 1 && n < a.axes && 2 * p >= first + a.sec[n - 1]) { first += a.sec[n - 1]; axis = n; at = place[n]; }
            if (!INTER) {
                int sec = a.sec[0];
#pragma unroll
                for (int n = 1; n < MVIT_ROTARY_AXES; ++n) sec = axis == n ? a.sec[n] : sec;
                ca = first + (p0 - first / 2);
                cb = ca + sec / 2;
            }
        }
        const double turn = at * a.turns[p];
        rot_sincos((float)(turn - __builtin_rint(turn)), sn[j], cs[j]);
        sn[j] *= a.sign;
    }
    int64_t bi = b, h = h0;
    for (int row = r0; row < r1; ++row) {
        const T* xh = x0 + bi * t.xs[0] + h * t.xs[1];
        T* yh = y0 + bi * t.ys[0] + h * t.ys[1];
        float u[V], w[V];
        rot_load_pair<T, V, INTER>(xh, ca, cb, u, w);
        float yu[V], yw[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (INTER) {                    // flat channel 2j, 2j + 1 of the 2 V in (u, w)
                const float xa = 2 * j < V ? u[(2 * j) % V] : w[(2 * j) % V];
                const float xb = 2 * j + 1 < V ? u[(2 * j + 1) % V] : w[(2 * j + 1) % V];
                const float ya = xa * cs[j] - xb * sn[j], yb = xa * sn[j] + xb * cs[j];
                if (2 * j < V) yu[(2 * j) % V] = ya; else yw[(2 * j) % V] = ya;
                if (2 * j + 1 < V) yu[(2 * j + 1) % V] = yb; else yw[(2 * j + 1) % V] = yb;
            } else {
                yu[j] = u[j] * cs[j] - w[j] * sn[j];
                yw[j] = u[j] * sn[j] + w[j] * cs[j];
            }
        }
        if (add0) {
            rot_load_pair<T, V, INTER>(add0 + bi * t.as[0] + h * t.as[1], ca, cb, u, w);
#pragma unroll
            for (int j = 0; j < V; ++j) { yu[j] += u[j]; yw[j] += w[j]; }
        }
        rot_store_pair<T, V, INTER>(yh, ca, cb, yu, yw);
        if (++h == t.H) { h = 0; ++bi; }
    }
}

template <typename T, int V>
static void rotary_launch(const RotaryArgs& a, uint32_t blocks, int layout, hipStream_t st) {
    if (layout) hipLaunchKernelGGL((rotary_kernel<T, V, true>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, V, false>), dim3(blocks), dim3(256), 0, st, a);
}

// ---- host side: whether two tensors [B][H][L][dim] share an element ------------------------------------------------------------------------
// Their extents may interleave (heads of one fused buffer), so the question is whether indices exist whose addresses are equal: a sum of strides
// times bounded whole numbers, searched from the largest stride down within what the smaller ones can still make up.
struct RotView {
    int64_t at;                    // address in elements
    int64_t n[3], s[3], dim;
    bool same(const RotView& o) const {
        for (int d = 0; d < 3; ++d)
            if (n[d] != o.n[d] || (n[d] > 1 && s[d] != o.s[d])) return false;
        return at == o.at;
    }
};
struct RotSum {
    enum { MOST = 7 };
    int64_t s[MOST], lo[MOST], hi[MOST], rest_lo[MOST + 1], rest_hi[MOST + 1];   // stride, least and most it is taken; what those behind make up
    int n = 0, budget = 0;
    void add(int64_t stride, int64_t low, int64_t high) {
        if (stride < 0) { stride = -stride; std::swap(low, high); low = -low; high = -high; }
        if (stride == 0) return;
        int i = 0;
        while (i < n && s[i] != stride) ++i;
        if (i == n) { s[n] = stride; lo[n] = hi[n] = 0; ++n; }
        lo[i] += low;
        hi[i] += high;
    }
    // may answer true where the budget ends, never false where there is a way
    bool makes(int64_t sum) {
        for (int i = 1; i < n; ++i)                      // largest stride first
            for (int j = i; j > 0 && s[j] > s[j - 1]; --j) { std::swap(s[j], s[j - 1]); std::swap(lo[j], lo[j - 1]); std::swap(hi[j], hi[j - 1]); }
        rest_lo[n] = rest_hi[n] = 0;
        for (int i = n - 1; i >= 0; --i) { rest_lo[i] = rest_lo[i + 1] + s[i] * lo[i]; rest_hi[i] = rest_hi[i + 1] + s[i] * hi[i]; }
        budget = 2000;
        return from(0, sum);
    }
    static int64_t down(int64_t a, int64_t b) { return a / b - (a % b != 0 && a < 0); }      // floor of a / b, b > 0
    bool from(int i, int64_t left) {
        if (left < rest_lo[i] || left > rest_hi[i]) return false;
        if (i == n || --budget < 0) return true;
        const int64_t a = std::max(lo[i], -down(rest_hi[i + 1] - left, s[i])), b = std::min(hi[i], down(left - rest_lo[i + 1], s[i]));
        for (int64_t k = a; k <= b; ++k)
            if (from(i + 1, left - k * s[i])) return true;
        return false;
    }
};
static bool rot_meet(const RotView& x, const RotView& y) {
    RotSum t;
    t.add(1, 1 - y.dim, x.dim - 1);
    for (int d = 0; d < 3; ++d) {
        t.add(x.s[d], 0, x.n[d] - 1);
        t.add(y.s[d], 1 - y.n[d], 0);
    }
    if (!t.makes(y.at - x.at)) return false;
    if (t.budget >= 0) return true;
    // Too many ways to try (every fourth token of a buffer beside all of them).  With the strides that are multiples of one of them counted as
    // that one, more sums can be made, not fewer: if there is no way then, there is none.
    for (int g = 0; g < t.n; ++g) {
        RotSum m;
        for (int i = 0; i < t.n; ++i) {
            const int64_t f = t.s[g] > 1 && t.s[i] % t.s[g] == 0 ? t.s[i] / t.s[g] : 1;
            m.add(t.s[i] / f, t.lo[i] * f, t.hi[i] * f);
        }
        if (!m.makes(y.at - x.at)) return false;
    }
    return true;
}
// two indices of one tensor name one element: not where every stride spans all that lies within it
static bool rot_meets_itself(const RotView& v) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return std::abs(v.s[i]) < std::abs(v.s[j]); });
    int64_t extent = v.dim;
    for (int d : order) {
        if (v.n[d] == 1) continue;
        if (std::abs(v.s[d]) < extent) return true;
        extent += (v.n[d] - 1) * std::abs(v.s[d]);
    }
    return false;
}

extern "C" int mvit_rotary_overlap(const mvit_rotary_tensor* tensors, int ntensors, int dim, int act_dtype) {
    if (!tensors || ntensors < 1 || ntensors > 2 || dim < 1) return MVIT_EINVAL;
    if (act_dtype != MVIT_F32 && act_dtype != MVIT_BF16) return MVIT_EDTYPE;
    const int64_t itemsize = act_dtype == MVIT_F32 ? 4 : 2;
    RotView v[2][3];               // x, y, add
    bool there[2][3] = {};
    for (int i = 0; i < ntensors; ++i) {
        const mvit_rotary_tensor& t = tensors[i];
        if (t.B <= 0 || t.H <= 0 || t.L <= 0) continue;
        const void* at[3] = {t.x, t.y, t.add};
        const int64_t* strides[3] = {t.xs, t.ys, t.as};
        for (int k = 0; k < 3; ++k)
            if (at[k]) {
                there[i][k] = true;
                v[i][k] = {(int64_t)(reinterpret_cast<uintptr_t>(at[k]) / itemsize), {t.B, t.H, t.L}, {strides[k][0], strides[k][1], strides[k][2]}, dim};
            }
    }
    for (int i = 0; i < ntensors; ++i) {
        if (!there[i][1]) continue;
        if (rot_meets_itself(v[i][1])) return 1;
        for (int j = 0; j < ntensors; ++j)
            for (int k = 0; k < 3; ++k)
                if (there[j][k] && !(i == j && (k == 1 || v[i][1].same(v[j][k]))) && rot_meet(v[i][1], v[j][k])) return 1;
    }
    return 0;
}

extern "C" int mvit_rotary_tensor_bytes(void) { return (int)sizeof(mvit_rotary_tensor); }

extern "C" int mvit_rotary(const mvit_rotary_tensor* tensors, int ntensors, int dim, int axes, const int* sections, const double* turns,
                           int layout, int inverse, int act_dtype, void* stream) {
    if (!tensors || ntensors < 1 || ntensors > 2 || dim < 1 || axes < 0 || axes > MVIT_ROTARY_AXES || (axes && (!sections || !turns)) ||
        (layout & ~1))
        return MVIT_EINVAL;
    if (act_dtype != MVIT_F32 && act_dtype != MVIT_BF16) return MVIT_EDTYPE;
    RotaryArgs a;
    a.dim = dim;
    a.axes = axes;
    a.sign = inverse ? -1.0f : 1.0f;
    const int itemsize = act_dtype == MVIT_F32 ? 4 : 2;
    int channels = 0;
    uint64_t fit = 16 / itemsize;           // a power of two: what every extent below has to be a multiple of
    auto narrow = [&fit](uint64_t v) { while (fit > 1 && v % fit) fit >>= 1; };
    for (int n = 0; n < MVIT_ROTARY_AXES; ++n) {
        a.sec[n] = n < axes ? sections[n] : 0;
        if (n < axes && (sections[n] < 2 || sections[n] % 2)) return MVIT_EINVAL;
        channels += a.sec[n];
        // pairs (i, i + s/2): a vector stays in its half, and every half begins at a multiple of it.  Interleaved pairs: only the sum counts
        if (!layout && n < axes) narrow(a.sec[n] / 2);
    }
    if (channels > dim || channels / 2 > MVIT_ROTARY_PAIRS) return MVIT_EINVAL;
    a.pairs = channels / 2;
    for (int p = 0; p < a.pairs; ++p) a.turns[p] = turns[p];
    narrow(a.pairs);
    narrow(dim - channels);
    uint64_t total_blocks = 0;
    for (int i = 0; i < 2; ++i) {
        a.first_block_1 = (uint32_t)total_blocks;
        a.blocks_per_group[i] = 1; a.groups[i] = 1; a.rows_per_thread[i] = 1; a.span[i] = 1;
        if (i >= ntensors) { a.t[i] = a.t[0]; a.first_block_1 = 0xffffffffu; continue; }
        const mvit_rotary_tensor& t = a.t[i] = tensors[i];
        if (t.B < 0 || t.H < 0 || t.L < 0) return MVIT_EINVAL;
        if (t.B == 0 || t.H == 0 || t.L == 0) continue;
        if (!t.x || !t.y || (t.pos && (t.pos_type < MVIT_POS_I32 || t.pos_type > MVIT_POS_F32))) return MVIT_EINVAL;
        if (!t.pos && axes) {
            int64_t n = 1;
            for (int k = 0; k < axes; ++k) {
                if (t.grid[k] < 1) return MVIT_EINVAL;
                n *= t.grid[k];
                if (n > t.L) return MVIT_EINVAL;
            }
            if (n != t.L) return MVIT_EINVAL;
        }
        const void* ptrs[3] = {t.x, t.y, t.add};
        const int64_t* strides[3] = {t.xs, t.ys, t.as};
        const int64_t extent[3] = {t.B, t.H, t.L};
        for (int k = 0; k < 3; ++k) {
            if (!ptrs[k]) continue;
            if (reinterpret_cast<uintptr_t>(ptrs[k]) % itemsize) return MVIT_EINVAL;
            narrow(reinterpret_cast<uintptr_t>(ptrs[k]) / itemsize);
            for (int d = 0; d < 3; ++d)     // (the stride of a single row is never used)
                if (extent[d] > 1) narrow((uint64_t)(strides[k][d] < 0 ? -strides[k][d] : strides[k][d]));
        }
    }
    if (mvit_rotary_overlap(tensors, ntensors, dim, act_dtype)) return MVIT_EINVAL;
    a.tasks = a.pairs / (int)fit + (dim - channels + 2 * (int)fit - 1) / (2 * (int)fit);
    // Rows per thread, so that a turn and its addresses serve several: until a thread moves 64 bytes each way (two rows of 16-byte vectors, at
    // most 8), as long as that leaves 1024 workgroups, four for each of the 256 CUs.  (1, 2, 4, 8 rows: one bf16 head on 8 x 112 x 112,
    // B = 8, 71, 62.7, 65.7, 68.5 us, in fp32 108, 112, 117, 122; 16 fp16 heads of 20011 listed tokens 163, 129, 129, 131; 8-byte vectors of four
    // heads on 8 x 28 x 28 20.5, 14.5, 13.4, 13.4; fp32 pairs by themselves 51, 37.7, 32.6, 29.4.  With 2048 / 1024 / 512 workgroups left: 19.0 / 18.5 /
    // 18.8.  The loads of two or four rows ahead of their stores: 62 to 176 us where one by one takes 63 to 131.)
    const int most = std::min(8, 32 / ((int)fit * itemsize));
    for (int i = 0; i < ntensors; ++i) {
        const mvit_rotary_tensor& t = a.t[i];
        if (i == 1) a.first_block_1 = (uint32_t)total_blocks;
        if (t.B == 0 || t.H == 0 || t.L == 0) continue;
        const uint64_t items = (uint64_t)t.L * a.tasks;
        if (items > 0xffffff00u || (int64_t)t.B * t.H > 0x7fffffff) return MVIT_EUNSUPPORTED;
        const uint64_t per = (items + 255) / 256;
        const bool shared = !t.pos || t.ps[0] == 0;
        const int span = shared ? t.B * t.H : t.H, spans = shared ? 1 : t.B;
        int rpt = 1;
        while (rpt < most && rpt < span && per * spans * (uint64_t)((span + 2 * rpt - 1) / (2 * rpt)) >= 1024) rpt *= 2;
        a.rows_per_thread[i] = rpt;
        a.span[i] = span;
        a.groups[i] = (uint32_t)((span + rpt - 1) / rpt);
        a.blocks_per_group[i] = (uint32_t)per;
        total_blocks += per * a.groups[i] * (uint64_t)spans;
        if (total_blocks > 0x7fffffffu) return MVIT_EUNSUPPORTED;
    }
    if (!total_blocks) return MVIT_OK;
    const uint32_t blocks = (uint32_t)total_blocks;
    hipStream_t st = as_stream(stream);
    if (act_dtype == MVIT_F32) {
        if (fit == 4) rotary_launch<float, 4>(a, blocks, layout, st);
        else if (fit == 2) rotary_launch<float, 2>(a, blocks, layout, st);
        else rotary_launch<float, 1>(a, blocks, layout, st);
    } else {
        if (fit == 8) rotary_launch<bf16_t, 8>(a, blocks, layout, st);
        else if (fit == 4) rotary_launch<bf16_t, 4>(a, blocks, layout, st);
        else if (fit == 2) rotary_launch<bf16_t, 2>(a, blocks, layout, st);
        else rotary_launch<bf16_t, 1>(a, blocks, layout, st);
    }
    MVIT_LAUNCH_CHECK();
    return MVIT_OK;
}
