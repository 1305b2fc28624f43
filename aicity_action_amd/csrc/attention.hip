// Fused pooled attention, head_dim 96:  O = softmax(q k^T * scale) v (+ q), scores never leave the CU.
//
// bf16 path (MFMA 32x32x16): one wave = 32 queries, 4 waves per workgroup, 64-key tiles.
//   S^T = K . Q^T   (A = K rows from LDS via ds_read_b128, B = Q^T held in registers) puts a QUERY on
//   each lane and 16 keys in its accumulator registers, so the softmax row reductions are in-register
//   (+ one cross-half exchange) and the exponentiated tile is already the B operand of
//   O^T += V^T . P^T (A = V^T read from a row-major V tile with ds_read_b64_tr_b16).
// fp32 path: exact-fp32 VALU kernel, one query per thread (parity path).
#include "common.h"

#define A_KT 64           // keys per tile
#define A_ROWB 192        // bytes per K/V row in LDS (96 bf16)
#define A_QW 32           // queries per wave
#define A_QB 128          // queries per workgroup

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((address_space(1))) const void a_gptr_t;
typedef __attribute__((address_space(3))) void a_lptr_t;
#define A_STAGES 3        // K/V tile ring (LDS-DMA, two tiles in flight)
#define A_TILEB (2 * A_KT * A_ROWB)   // K image + V image of one tile = 24 KiB

__device__ __forceinline__ int kslab_off(int row, int chunk) {
    int p = chunk + ((row >> 2) & 3);
    p = p >= 12 ? p - 12 : p;
    return row * A_ROWB + p * 16;
}

// Transposed LDS read issued as inline asm: through the builtin the compiler cannot tell the read apart from the
// in-flight LDS-DMA writes of later tiles and puts s_waitcnt vmcnt(0) in front of it, which serialises the K/V ring.
// The caller waits with lds_tr_wait() (operands tie the registers to the wait) before the first use.
template <int OFF>
__device__ __forceinline__ bf16x4 lds_tr16(uint32_t addr) {
    bf16x4 v;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
    return v;
}

template <bool ADD_Q, int NW>      // NW waves x 32 queries per workgroup
__global__ __launch_bounds__(64 * NW) void attn_fwd_bf16_kernel(const bf16_t* __restrict__ Q, const bf16_t* __restrict__ Kt,
                                                            const bf16_t* __restrict__ V, bf16_t* __restrict__ O,
                                                            float* __restrict__ LSE, int heads, int Lq, int Lk,
                                                            float scale_log2e) {
    extern __shared__ __attribute__((aligned(16))) char smem[];   // A_STAGES x (K image 12 KiB | V image 12 KiB)

    int qtile, bh;                        // bh = b*heads + g
    xcd_group_map(qtile, bh);
    const int b = bh / heads, g = bh - b * heads;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int r = lane & 31, h = lane >> 5;
    const int q0 = qtile * (A_QW * NW) + wave * A_QW;

    const bf16_t* Qb = Q + (int64_t)bh * Lq * 96;
    const bf16_t* Kb = Kt + (int64_t)bh * Lk * 96;
    const bf16_t* Vb = V + (int64_t)bh * Lk * 96;

    // Q^T fragments: lane (r,h) holds Q[q0+r][16ks + 8h .. +7]
    int qi = q0 + r;
    const bool q_ok = qi < Lq;
    qi = q_ok ? qi : Lq - 1;
    bf16x8 qf[6];
#pragma unroll
    for (int ks = 0; ks < 6; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(Qb + (int64_t)qi * 96 + 16 * ks + 8 * h);

    // K/V tiles go global -> LDS by DMA (global_load_lds_dwordx4: 64 lanes x 16 B land linearly at a wave-uniform LDS
    // base): the 24 pieces of 1 KiB of a tile (12 of the K image, then 12 of the V image) are dealt PW = 24/NW per wave, so a
    // wave moves only K or only V.  A tile is one contiguous 12 KiB block of K (and V); LDS position p = 64*piece + lane of the
    // K image holds chunk (p%12 - rot(row)) of row p/12, so the rotation swizzle is applied to the SOURCE address; the V image
    // is linear.  Nothing is staged in registers.
    constexpr int PW = 24 / NW;
    const bool is_v = wave >= NW / 2;                       // wave-uniform
    const char* src_bh = reinterpret_cast<const char*>(is_v ? Vb : Kb);
    uint32_t g_off[PW];
    int p_row[PW], p_c[PW];
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int piece = PW * wave + i - (is_v ? 12 : 0);
        const int p = 64 * piece + lane;
        const int row = p / 12, pos = p - row * 12;
        int c = pos;
        if (!is_v) {
            c = pos - ((row >> 2) & 3);
            c = c < 0 ? c + 12 : c;
        }
        p_row[i] = row; p_c[i] = c;
        g_off[i] = (uint32_t)(row * 12 + c) * 16u;
    }
    auto dma = [&](int k0, int stage) {
        const char* t_base = src_bh + (int64_t)k0 * A_ROWB;   // wave-uniform
        char* dst = smem + stage * A_TILEB + 1024 * (PW * wave);
        if (k0 + A_KT <= Lk) {
#pragma unroll
            for (int i = 0; i < PW; ++i)
                __builtin_amdgcn_global_load_lds((a_gptr_t*)(t_base + g_off[i]), (a_lptr_t*)(dst + 1024 * i), 16, 0, 0);
        } else {        // tail tile: rows past Lk re-read the last valid row (finite data; their scores are masked to -inf)
            const int last = Lk - 1 - k0;
#pragma unroll
            for (int i = 0; i < PW; ++i) {
                const int row = p_row[i] < last ? p_row[i] : last;
                __builtin_amdgcn_global_load_lds((a_gptr_t*)(t_base + (uint32_t)(row * 12 + p_c[i]) * 16u), (a_lptr_t*)(dst + 1024 * i), 16, 0, 0);
            }
        }
    };

    int koff[6];  // K fragment chunk offsets for this lane
#pragma unroll
    for (int ks = 0; ks < 6; ++ks) {
        int p = 2 * ks + h + ((r >> 2) & 3);
        p = p >= 12 ? p - 12 : p;
        koff[ks] = p * 16;
    }
    // transposed V read: lane supplies the address of key-row (4h + q) and d columns 16*(gi&1) + 4p
    const int i16 = lane & 15, gi = lane >> 4;
    const int v_lane_off = (4 * h + (i16 >> 2)) * A_ROWB + (16 * (gi & 1) + 4 * (i16 & 3)) * 2;

    f32x16 o[3];
#pragma unroll
    for (int db = 0; db < 3; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    const int nkt = (Lk + A_KT - 1) / A_KT;
    dma(0, 0);
    if (nkt > 1) dma(A_KT, 1);
    // consume the Q fragments once here: the vmcnt wait for them is paid before the loop, so inside it only the counted
    // waits below touch vmcnt (the K/V DMAs stay in flight under the MFMAs)
#pragma unroll
    for (int ks = 0; ks < 6; ++ks) asm volatile("" : "+v"(qf[ks]));
    int stage = 0;
#ifdef ATT_STAMP
    uint64_t tacc[6] = {0, 0, 0, 0, 0, 0};
    uint64_t tp = __builtin_readcyclecounter();
    const uint64_t t_begin = tp, w_begin = wall_clock64();
#define STAMP(i) { const uint64_t now_ = __builtin_readcyclecounter(); tacc[i] += now_ - tp; tp = now_; }
#else
#define STAMP(i)
#endif
    for (int kt = 0; kt < nkt; ++kt) {
        // tile kt has landed once at most the PW pieces of tile kt+1 are still outstanding (VMEM returns in order)
        if (kt + 1 < nkt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        STAMP(0)
        __builtin_amdgcn_s_barrier();       // everyone's pieces landed; everyone is done with the stage refilled below
        if (kt + 2 < nkt) dma((kt + 2) * A_KT, stage == 0 ? 2 : stage - 1);
        const char* sK = smem + stage * A_TILEB;
        const char* sV = sK + A_KT * A_ROWB;
        stage = stage == A_STAGES - 1 ? 0 : stage + 1;
        STAMP(1)

        // ---- S^T = K . Q^T  (two 32-key blocks) ------------------------------------------------
        f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
        {   // all 12 K fragments are requested before the first MFMA (counted lgkmcnt waits): LDS latency is paid once
            bf16x8 kf[6][2];
#pragma unroll
            for (int ks = 0; ks < 6; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    kf[ks][kb] = *reinterpret_cast<const bf16x8*>(sK + (32 * kb + r) * A_ROWB + koff[ks]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < 6; ++ks)       // the two key blocks alternate: no back-to-back dependent MFMAs
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) s[kb] = mfma16(kf[ks][kb], qf[ks], s[kb]);
            __builtin_amdgcn_sched_barrier(0);
        }
        // V^T fragments of the whole tile: requested now, they land under the softmax arithmetic
        bf16x4 vlo[12], vhi[12];
        {
            const uint32_t va = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)(sV) + v_lane_off;
#define VTR(S16, DB) vlo[3 * S16 + DB] = lds_tr16<S16 * 16 * A_ROWB + DB * 64>(va); vhi[3 * S16 + DB] = lds_tr16<S16 * 16 * A_ROWB + DB * 64 + 8 * A_ROWB>(va);
            VTR(0, 0) VTR(0, 1) VTR(0, 2) VTR(1, 0) VTR(1, 1) VTR(1, 2) VTR(2, 0) VTR(2, 1) VTR(2, 2) VTR(3, 0) VTR(3, 1) VTR(3, 2)
#undef VTR
        }
        // ---- online softmax: raw-score running max, scale folded into the exp2 argument -----------------
        const int kbase = kt * A_KT;
        if (kbase + A_KT > Lk) {           // tail tile only (wave-uniform): mask keys >= Lk
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = kbase + 32 * kb + (i & 3) + 8 * (i >> 2) + 4 * h;
                    s[kb][i] = key < Lk ? s[kb][i] : -INFINITY;
                }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, s[0][i]), s[1][i]);      // v_max3_f32
        {   // both halves of the wave hold the same 32 queries (different keys): exchange maxima
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        }
        STAMP(2)
        const float m_new = fmaxf(m_run, mx);
        if (__any(m_new > m_run)) {        // rescale only when some query's running max moved
            const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * scale_log2e);
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < 3; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
            m_run = m_new;
        }
        const f32x2 c2 = {scale_log2e, scale_log2e};
        const float mcs = -m_run * scale_log2e;
        const f32x2 mc2 = {mcs, mcs};
        f32x2 ps2 = {0.f, 0.f};
        bf16x8 pf[4];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int sh = 0; sh < 2; ++sh) {
                uint32_t pk[4];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const f32x2 sv = {s[kb][8 * sh + 2 * jj], s[kb][8 * sh + 2 * jj + 1]};
                    const f32x2 t = __builtin_elementwise_fma(sv, c2, mc2);
                    const f32x2 pp = {__builtin_amdgcn_exp2f(t[0]), __builtin_amdgcn_exp2f(t[1])};
                    ps2 += pp;
                    pk[jj] = pack_bf16x2(pp[0], pp[1]);
                }
                uint4 u = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                pf[2 * kb + sh] = *reinterpret_cast<bf16x8*>(&u);
            }
        const float psum = ps2[0] + ps2[1];
        l_run += psum;
        STAMP(3)
        // ---- O^T += V^T . P^T -------------------------------------------------------------------
        asm volatile("s_waitcnt lgkmcnt(0)"
                     : "+v"(vlo[0]), "+v"(vlo[1]), "+v"(vlo[2]), "+v"(vlo[3]), "+v"(vlo[4]), "+v"(vlo[5]), "+v"(vlo[6]), "+v"(vlo[7]),
                       "+v"(vlo[8]), "+v"(vlo[9]), "+v"(vlo[10]), "+v"(vlo[11]));
        asm volatile("" : "+v"(vhi[0]), "+v"(vhi[1]), "+v"(vhi[2]), "+v"(vhi[3]), "+v"(vhi[4]), "+v"(vhi[5]), "+v"(vhi[6]), "+v"(vhi[7]),
                          "+v"(vhi[8]), "+v"(vhi[9]), "+v"(vhi[10]), "+v"(vhi[11]));
#pragma unroll
        for (int s16 = 0; s16 < 4; ++s16) {
#pragma unroll
            for (int db = 0; db < 3; ++db) {
                const bf16x4 lo = vlo[3 * s16 + db], hi = vhi[3 * s16 + db];
                bf16x8 vf;
                vf[0] = lo[0]; vf[1] = lo[1]; vf[2] = lo[2]; vf[3] = lo[3];
                vf[4] = hi[0]; vf[5] = hi[1]; vf[6] = hi[2]; vf[7] = hi[3];
                o[db] = mfma16(vf, pf[s16], o[db]);
            }
        }
        STAMP(4)
    }
#ifdef ATT_STAMP
    if (LSE && lane == 0) {
        for (int i = 0; i < 6; ++i) LSE[(int64_t)bh * Lq + qtile * A_QB + wave * 8 + i] = (float)tacc[i] / nkt;
        LSE[(int64_t)bh * Lq + qtile * A_QB + wave * 8 + 6] = (float)(__builtin_readcyclecounter() - t_begin);
        LSE[(int64_t)bh * Lq + qtile * A_QB + wave * 8 + 7] = (float)(wall_clock64() - w_begin);
        return;
    }
#endif
    // ---- epilogue: normalise, + q residual, store [b][q][g*96 + d] -------------------------------
    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = 1.0f / l_tot;
    if (LSE && q_ok && h == 0) LSE[(int64_t)bh * Lq + qi] = m_run * scale_log2e + __builtin_amdgcn_logf(l_tot);  // log2 domain
    if (q_ok) {
        const int C = heads * 96;
        bf16_t* orow = O + ((int64_t)b * Lq + qi) * C + g * 96;
        const bf16_t* qrow = Qb + (int64_t)qi * 96;
#pragma unroll
        for (int db = 0; db < 3; ++db)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const int d = 32 * db + 8 * i4 + 4 * h;
                float4 v = make_float4(o[db][4 * i4 + 0] * inv, o[db][4 * i4 + 1] * inv, o[db][4 * i4 + 2] * inv,
                                       o[db][4 * i4 + 3] * inv);
                if (ADD_Q) {
                    const float4 qq = load4(qrow + d);
                    v.x += qq.x; v.y += qq.y; v.z += qq.z; v.w += qq.w;
                }
                store4(orow + d, v);
            }
    }
}

// ------------------------------------------------------------------------------------------------
// Software-pipelined variant (4 waves x 32 queries): inside one wave the score MFMAs of tile t+1 are issued between the
// exponentials of tile t, and the running-max reduction of tile t+1 between the P.V MFMAs of tile t, so the matrix pipe
// and the VALU of a SIMD both have work from ONE wave (the two co-resident waves of different workgroups then fill each
// other's remaining gaps).  K runs one tile ahead of V: separate 3-deep LDS rings, K waves load tile t+3 while V waves
// load tile t+2, both with one older load still in flight behind the counted wait.
// ------------------------------------------------------------------------------------------------
#define AP_RING (3 * A_KT * A_ROWB)      // one ring (K or V): 3 x 12 KiB

template <int OFF>
__device__ __forceinline__ bf16x8 lds_rd128(uint32_t addr) {
    bf16x8 v;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
    return v;
}
#ifndef ATT_ABL
#define ATT_ABL 0      // timing ablations of tools/ab_attn_abl.sh (results invalid when non-zero)
#endif
#define AP_WAIT6(N, a, b, c, d, e, f) asm volatile("s_waitcnt lgkmcnt(%6)" : "+v"(a), "+v"(b), "+v"(c), "+v"(d), "+v"(e), "+v"(f) : "n"((ATT_ABL & 64) ? 15 : N))

// SLOT: every MFMA of regions R1..R4 is followed by its own small bundle of softmax VALU work, pinned by scheduling barriers
// (one exp2 pair = pk_fma, 2 exp, cvt_pk, pk_add per MFMA gap) instead of leaving the interleave to the compiler
template <bool ADD_Q, bool SLOT>
__global__ __launch_bounds__(256, 2) void attn_fwd_pipe_kernel(const bf16_t* __restrict__ Q, const bf16_t* __restrict__ Kt,
                                                               const bf16_t* __restrict__ V, bf16_t* __restrict__ O,
                                                               float* __restrict__ LSE, int heads, int Lq, int Lk,
                                                               float scale_log2e) {
    extern __shared__ __attribute__((aligned(16))) char smem[];   // K ring 36 KiB | V ring 36 KiB
    constexpr int NW = 4, PW = 6;

    int qtile, bh;
    xcd_group_map(qtile, bh);
    const int b = bh / heads, g = bh - b * heads;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int r = lane & 31, h = lane >> 5;
    const int q0 = qtile * (A_QW * NW) + wave * A_QW;

    const bf16_t* Qb = Q + (int64_t)bh * Lq * 96;
    const bf16_t* Kb = Kt + (int64_t)bh * Lk * 96;
    const bf16_t* Vb = V + (int64_t)bh * Lk * 96;

    int qi = q0 + r;
    const bool q_ok = qi < Lq;
    qi = q_ok ? qi : Lq - 1;
    bf16x8 qf[6];
#pragma unroll
    for (int ks = 0; ks < 6; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(Qb + (int64_t)qi * 96 + 16 * ks + 8 * h);

    const bool is_v = wave >= NW / 2;                       // wave-uniform: waves 0,1 move K tiles, waves 2,3 V tiles
    const char* src_bh = reinterpret_cast<const char*>(is_v ? Vb : Kb);
    // piece i of this wave covers LDS positions p = 64*(PW*(wave&1) + i) + lane of the 12-KiB tile image: row p/12, 16-B slot
    // p%12, which holds source chunk (slot - rot(row)) mod 12 for K (rotation swizzle on the SOURCE address) and chunk = slot
    // for V.  Pieces i and i+3 are exactly 16 rows apart (same rotation), so three lane offsets + an immediate serve all six.
    auto piece_off = [&](int i, int ln, int last_row) -> uint32_t {
        const int p = 64 * (PW * (wave & 1) + i) + ln;
        int row = p / 12, c = p - row * 12;
        if (!is_v) {
            c -= (row >> 2) & 3;
            c = c < 0 ? c + 12 : c;
        }
        row = row < last_row ? row : last_row;
        return (uint32_t)(row * 12 + c) * 16u;
    };
    uint32_t g_off[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) g_off[i] = piece_off(i, lane, A_KT);
    const uint32_t smem_a = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)(smem);
    const uint32_t ring_a = smem_a + (is_v ? AP_RING : 0) + 1024 * (PW * (wave & 1));
    // the DMA is issued as inline asm (SGPR base + 32-bit lane offset, LDS base in M0): through the builtin the compiler keeps
    // 64-bit lane addresses in registers across the loop, spills them, and waits vmcnt(0) on the reloads between the pieces
    auto dma1 = [&](const char* base, uint32_t off, uint32_t lds) {
        // (M0 cannot be named as a clobber; nothing else in this kernel depends on it: gfx9+ LDS instructions do not read M0)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
    };
    auto dma = [&](int tile, int stage) {
        const int k0 = tile * A_KT;
        const char* t_base = src_bh + (int64_t)k0 * A_ROWB;   // wave-uniform
        const uint32_t dst = __builtin_amdgcn_readfirstlane(ring_a + stage * (A_KT * A_ROWB));
        if (k0 + A_KT <= Lk) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                dma1(t_base, g_off[i], dst + 1024 * i);
                dma1(t_base + 16 * A_ROWB, g_off[i], dst + 1024 * (i + 3));
            }
        } else {        // tail tile: rows past Lk re-read the last valid row (finite data; their scores are masked to -inf)
            int ln = lane;
            asm volatile("" : "+v"(ln));      // keeps this rare path's address arithmetic inside the branch (not hoisted into loop-long registers)
#pragma unroll
            for (int i = 0; i < PW; ++i) dma1(t_base, piece_off(i, ln, Lk - 1 - k0), dst + 1024 * i);
        }
    };

    // K fragment of k-step ks: row r, 16-B chunk (2ks + h + rot(r)) mod 12 with rot <= 3: k-steps 0..3 never wrap (immediate
    // offsets from one lane address), k-steps 4 and 5 each get their own
    uint32_t ka0, ka4, ka5;
    {
        const int p0 = h + ((r >> 2) & 3);
        const int p4 = p0 + 8 >= 12 ? p0 + 8 - 12 : p0 + 8, p5 = p0 + 10 >= 12 ? p0 + 10 - 12 : p0 + 10;
        ka0 = smem_a + r * A_ROWB + p0 * 16;
        ka4 = smem_a + r * A_ROWB + p4 * 16;
        ka5 = smem_a + r * A_ROWB + p5 * 16;
    }
    const int i16 = lane & 15, gi = lane >> 4;
    const uint32_t va0 = smem_a + AP_RING + (4 * h + (i16 >> 2)) * A_ROWB + (16 * (gi & 1) + 4 * (i16 & 3)) * 2;

    f32x16 o[3];
#pragma unroll
    for (int db = 0; db < 3; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run, l_run = 0.f;

    const int nkt = (Lk + A_KT - 1) / A_KT;
    // prologue loads: K tiles 0,1,2 / V tiles 0,1
    dma(0, 0);
    if (nkt > 1) dma(1, 1);
    if (!is_v && nkt > 2) dma(2, 2);
#pragma unroll
    for (int ks = 0; ks < 6; ++ks) asm volatile("" : "+v"(qf[ks]));

    // masks keys >= Lk of the (last) tile kt in a score tile, then the row maximum over the tile (both wave halves)
    auto tile_max = [&](f32x16 (&s)[2], int kt) -> float {
        const int kbase = kt * A_KT;
        if (kbase + A_KT > Lk) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = kbase + 32 * kb + (i & 3) + 8 * (i >> 2) + 4 * h;
                    s[kb][i] = key < Lk ? s[kb][i] : -INFINITY;
                }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, s[0][i]), s[1][i]);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    };

#define AP_KRD(KF, KS, KA, OFF) if (!(ATT_ABL & 32)) { KF[KS][0] = lds_rd128<OFF>(KA); KF[KS][1] = lds_rd128<OFF + 32 * A_ROWB>(KA); }
#define AP_VTR(VL, VH, S16, DB, VA) if (!(ATT_ABL & 32)) VL[3 * (S16 & 1) + DB] = lds_tr16<S16 * 16 * A_ROWB + DB * 64>(VA); if (!(ATT_ABL & 32)) VH[3 * (S16 & 1) + DB] = lds_tr16<S16 * 16 * A_ROWB + DB * 64 + 8 * A_ROWB>(VA);
#define AP_EXP(S, KB, SH) if (ATT_ABL & 1) { \
        uint4 u_ = make_uint4(__float_as_uint(S[KB][8 * SH]), __float_as_uint(S[KB][8 * SH + 2]), __float_as_uint(S[KB][8 * SH + 4]), __float_as_uint(S[KB][8 * SH + 6])); \
        pf[2 * KB + SH] = *reinterpret_cast<bf16x8*>(&u_); } else { \
        uint32_t pk_[4]; \
        _Pragma("unroll") for (int jj = 0; jj < 4; ++jj) { \
            const f32x2 sv_ = {S[KB][8 * SH + 2 * jj], S[KB][8 * SH + 2 * jj + 1]}; \
            const f32x2 t_ = __builtin_elementwise_fma(sv_, c2, mc2); \
            const f32x2 pp_ = {__builtin_amdgcn_exp2f(t_[0]), __builtin_amdgcn_exp2f(t_[1])}; \
            ps2 += pp_; \
            pk_[jj] = pack_bf16x2(pp_[0], pp_[1]); \
        } \
        uint4 u_ = make_uint4(pk_[0], pk_[1], pk_[2], pk_[3]); \
        pf[2 * KB + SH] = *reinterpret_cast<bf16x8*>(&u_); }
#define AP_PAIR(S, KB, SH, JJ) { \
        const f32x2 sv_ = {S[KB][8 * SH + 2 * JJ], S[KB][8 * SH + 2 * JJ + 1]}; \
        const f32x2 t_ = __builtin_elementwise_fma(sv_, c2, mc2); \
        const f32x2 pp_ = {__builtin_amdgcn_exp2f(t_[0]), __builtin_amdgcn_exp2f(t_[1])}; \
        ps2 += pp_; \
        pkw[2 * KB + SH][JJ] = pack_bf16x2(pp_[0], pp_[1]); }
#define AP_PFIN(E) { uint4 u_ = make_uint4(pkw[E][0], pkw[E][1], pkw[E][2], pkw[E][3]); pf[E] = *reinterpret_cast<bf16x8*>(&u_); }
#define AP_SB __builtin_amdgcn_sched_barrier(0);
#define AP_PV1(VL, VH, S16, DB) { \
        const bf16x4 lo_ = VL[3 * (S16 & 1) + DB], hi_ = VH[3 * (S16 & 1) + DB]; \
        bf16x8 vf_; \
        vf_[0] = lo_[0]; vf_[1] = lo_[1]; vf_[2] = lo_[2]; vf_[3] = lo_[3]; vf_[4] = hi_[0]; vf_[5] = hi_[1]; vf_[6] = hi_[2]; vf_[7] = hi_[3]; \
        o[DB] = mfma16(vf_, pf[S16], o[DB]); }
#define AP_MX4(I0) mx = fmaxf(fmaxf(mx, nx[0][I0]), nx[1][I0]); mx = fmaxf(fmaxf(mx, nx[0][I0 + 1]), nx[1][I0 + 1]); \
        mx = fmaxf(fmaxf(mx, nx[0][I0 + 2]), nx[1][I0 + 2]); mx = fmaxf(fmaxf(mx, nx[0][I0 + 3]), nx[1][I0 + 3]);
// scheduling pattern for a region of NM MFMAs: NV VALU instructions after each MFMA (the rest follow the last one)
#define AP_MIX(NM, NV) _Pragma("unroll") for (int i_ = 0; i_ < NM; ++i_) { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, NV, 0); }
#define AP_PV(VL, VH, S16) _Pragma("unroll") for (int db = 0; db < 3; ++db) { \
        const bf16x4 lo_ = VL[3 * (S16 & 1) + db], hi_ = VH[3 * (S16 & 1) + db]; \
        bf16x8 vf_; \
        vf_[0] = lo_[0]; vf_[1] = lo_[1]; vf_[2] = lo_[2]; vf_[3] = lo_[3]; vf_[4] = hi_[0]; vf_[5] = hi_[1]; vf_[6] = hi_[2]; vf_[7] = hi_[3]; \
        if (!(ATT_ABL & 16)) o[db] = mfma16(vf_, pf[S16], o[db]); }

    int kst = 0, vst = 0;     // ring stage of K tile kt+1 / V tile kt (set below)
    f32x16 sa[2], sb[2];
    {   // ---- prologue: S(0) and its row maximum --------------------------------------------------
        if (nkt > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PW) : "memory");
        else if (nkt > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        bf16x8 kf[6][2];
        AP_KRD(kf, 0, ka0, 0) AP_KRD(kf, 1, ka0, 32) AP_KRD(kf, 2, ka0, 64) AP_KRD(kf, 3, ka0, 96) AP_KRD(kf, 4, ka4, 0) AP_KRD(kf, 5, ka5, 0)
        AP_WAIT6(0, kf[0][0], kf[0][1], kf[1][0], kf[1][1], kf[2][0], kf[2][1]);
        asm volatile("" : "+v"(kf[3][0]), "+v"(kf[3][1]), "+v"(kf[4][0]), "+v"(kf[4][1]), "+v"(kf[5][0]), "+v"(kf[5][1]));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sa[kb][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 6; ++ks)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) sa[kb] = mfma16(kf[ks][kb], qf[ks], sa[kb]);
        m_run = tile_max(sa, 0);
        kst = 1;
    }

    // one tile: P(kt) from `cur`, O += V(kt)^T P(kt); with NEXT also S(kt+1) -> `nx` and the running-max update
    auto step = [&](f32x16 (&cur)[2], f32x16 (&nx)[2], int kt, auto next_tag) {
        constexpr bool NEXT = decltype(next_tag)::value;
        // K(kt+1) (K waves) / V(kt) (V waves) landed once at most the newest load of this wave is outstanding
        if (ATT_ABL & 128) {}
        else if (kt + 2 < nkt) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (!(ATT_ABL & 4)) __builtin_amdgcn_s_barrier();
        {   // refill the stage everyone has left: K tile kt+3 replaces K(kt), V tile kt+2 replaces V(kt-1)
            const int t_new = kt + (is_v ? 2 : 3);
            if (!(ATT_ABL & 2) && t_new < nkt) dma(t_new, is_v ? (vst == 0 ? 2 : vst - 1) : (kst == 0 ? 2 : kst - 1));
        }
        const uint32_t k_base = kst * (A_KT * A_ROWB), v_addr = va0 + vst * (A_KT * A_ROWB);
        kst = kst == 2 ? 0 : kst + 1;
        vst = vst == 2 ? 0 : vst + 1;

        const f32x2 c2 = {scale_log2e, scale_log2e};
        const float mcs = -m_run * scale_log2e;
        const f32x2 mc2 = {mcs, mcs};
        f32x2 ps2 = {0.f, 0.f};
        bf16x8 pf[4];
        uint32_t pkw[4][4];
        bf16x8 kf[3][2];
        bf16x4 vl[6], vh[6];
        // LDS reads return in order: each region requests the operands of the NEXT matrix region, then waits (counted) for its own
        // R0: K(kt+1) k-steps 0..2 requested; first 16 keys of P
        if (NEXT) {
            const uint32_t a0 = ka0 + k_base;
            AP_KRD(kf, 0, a0, 0) AP_KRD(kf, 1, a0, 32) AP_KRD(kf, 2, a0, 64)
        }
        AP_EXP(cur, 0, 0)
        __builtin_amdgcn_sched_barrier(0);
        // R1: V(kt) keys 0..15 requested; S(kt+1) k-steps 0..2 beside the next 16 keys of P
        AP_VTR(vl, vh, 0, 0, v_addr) AP_VTR(vl, vh, 0, 1, v_addr) AP_VTR(vl, vh, 0, 2, v_addr)
        if (NEXT) {
            AP_WAIT6(6, kf[0][0], kf[0][1], kf[1][0], kf[1][1], kf[2][0], kf[2][1]);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) nx[kb][i] = 0.f;
            if constexpr (SLOT) {
                nx[0] = mfma16(kf[0][0], qf[0], nx[0]); AP_PAIR(cur, 0, 1, 0) AP_SB
                nx[1] = mfma16(kf[0][1], qf[0], nx[1]); AP_PAIR(cur, 0, 1, 1) AP_SB
                nx[0] = mfma16(kf[1][0], qf[1], nx[0]); AP_PAIR(cur, 0, 1, 2) AP_SB
                nx[1] = mfma16(kf[1][1], qf[1], nx[1]); AP_PAIR(cur, 0, 1, 3) AP_SB
                nx[0] = mfma16(kf[2][0], qf[2], nx[0]); AP_SB
                nx[1] = mfma16(kf[2][1], qf[2], nx[1]); AP_PFIN(1) AP_SB
            } else {
#pragma unroll
            for (int ks = 0; ks < 3; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) if (!(ATT_ABL & 8)) nx[kb] = mfma16(kf[ks][kb], qf[ks], nx[kb]);
            }
        }
        if (!(SLOT && NEXT)) { AP_EXP(cur, 0, 1) }
        if (NEXT && !SLOT) { AP_MIX(6, 3) }
        __builtin_amdgcn_sched_barrier(0);
        // R2: V keys 16..31 and K(kt+1) k-steps 3..5 requested; O += V^T P over keys 0..31 beside the third 16 keys of P
        AP_VTR(vl, vh, 1, 0, v_addr) AP_VTR(vl, vh, 1, 1, v_addr) AP_VTR(vl, vh, 1, 2, v_addr)
        if (NEXT) {
            AP_KRD(kf, 0, ka0 + k_base, 96) AP_KRD(kf, 1, ka4 + k_base, 0) AP_KRD(kf, 2, ka5 + k_base, 0)
            AP_WAIT6(12, vl[0], vl[1], vl[2], vh[0], vh[1], vh[2]);
        } else {
            AP_WAIT6(6, vl[0], vl[1], vl[2], vh[0], vh[1], vh[2]);
        }
        if constexpr (SLOT) {
            AP_PV1(vl, vh, 0, 0) AP_PAIR(cur, 1, 0, 0) AP_SB
            AP_PV1(vl, vh, 0, 1) AP_PAIR(cur, 1, 0, 1) AP_SB
            AP_PV1(vl, vh, 0, 2) AP_PAIR(cur, 1, 0, 2) AP_SB
            if (NEXT) AP_WAIT6(6, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
            else AP_WAIT6(0, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
            AP_PV1(vl, vh, 1, 0) AP_PAIR(cur, 1, 0, 3) AP_SB
            AP_PV1(vl, vh, 1, 1) AP_SB
            AP_PV1(vl, vh, 1, 2) AP_PFIN(2) AP_SB
        } else {
        AP_PV(vl, vh, 0)
        if (NEXT) AP_WAIT6(6, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
        else AP_WAIT6(0, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
        AP_PV(vl, vh, 1)
        AP_EXP(cur, 1, 0)
        AP_MIX(6, 3)
        }
        __builtin_amdgcn_sched_barrier(0);
        // R3: V(kt) keys 32..47 requested; S(kt+1) k-steps 3..5 beside the last 16 keys of P
        AP_VTR(vl, vh, 2, 0, v_addr) AP_VTR(vl, vh, 2, 1, v_addr) AP_VTR(vl, vh, 2, 2, v_addr)
        if (NEXT) {
            AP_WAIT6(6, kf[0][0], kf[0][1], kf[1][0], kf[1][1], kf[2][0], kf[2][1]);
            if constexpr (SLOT) {
                nx[0] = mfma16(kf[0][0], qf[3], nx[0]); AP_PAIR(cur, 1, 1, 0) AP_SB
                nx[1] = mfma16(kf[0][1], qf[3], nx[1]); AP_PAIR(cur, 1, 1, 1) AP_SB
                nx[0] = mfma16(kf[1][0], qf[4], nx[0]); AP_PAIR(cur, 1, 1, 2) AP_SB
                nx[1] = mfma16(kf[1][1], qf[4], nx[1]); AP_PAIR(cur, 1, 1, 3) AP_SB
                nx[0] = mfma16(kf[2][0], qf[5], nx[0]); AP_SB
                nx[1] = mfma16(kf[2][1], qf[5], nx[1]); AP_PFIN(3) AP_SB
            } else {
#pragma unroll
            for (int ks = 0; ks < 3; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) if (!(ATT_ABL & 8)) nx[kb] = mfma16(kf[ks][kb], qf[ks + 3], nx[kb]);
            }
        }
        if (!(SLOT && NEXT)) { AP_EXP(cur, 1, 1) }
        if (NEXT && !SLOT) { AP_MIX(6, 3) }
        __builtin_amdgcn_sched_barrier(0);
        // R4: V keys 48..63 requested; O += V^T P over keys 32..63 beside the row maximum of S(kt+1)
        AP_VTR(vl, vh, 3, 0, v_addr) AP_VTR(vl, vh, 3, 1, v_addr) AP_VTR(vl, vh, 3, 2, v_addr)
        float mx = 0.f;
        if constexpr (SLOT && NEXT) {
            if ((kt + 2) * A_KT > Lk) {           // S(kt+1) is the (ragged) last tile: mask keys >= Lk (wave-uniform, once per kernel)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = (kt + 1) * A_KT + 32 * kb + (i & 3) + 8 * (i >> 2) + 4 * h;
                        nx[kb][i] = key < Lk ? nx[kb][i] : -INFINITY;
                    }
            }
            AP_WAIT6(6, vl[0], vl[1], vl[2], vh[0], vh[1], vh[2]);
            AP_PV1(vl, vh, 2, 0) AP_SB
            AP_PV1(vl, vh, 2, 1) mx = fmaxf(nx[0][0], nx[1][0]); mx = fmaxf(fmaxf(mx, nx[0][1]), nx[1][1]); mx = fmaxf(fmaxf(mx, nx[0][2]), nx[1][2]); mx = fmaxf(fmaxf(mx, nx[0][3]), nx[1][3]); AP_SB
            AP_PV1(vl, vh, 2, 2) AP_MX4(4) AP_SB
            AP_WAIT6(0, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
            AP_PV1(vl, vh, 3, 0) AP_MX4(8) AP_SB
            AP_PV1(vl, vh, 3, 1) AP_MX4(12) AP_SB
            AP_PV1(vl, vh, 3, 2)
            {
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            }
        } else {
        AP_WAIT6(6, vl[0], vl[1], vl[2], vh[0], vh[1], vh[2]);
        AP_PV(vl, vh, 2)
        AP_WAIT6(0, vl[3], vl[4], vl[5], vh[3], vh[4], vh[5]);
        AP_PV(vl, vh, 3)
        if (NEXT) mx = tile_max(nx, kt + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        l_run += ps2[0] + ps2[1];
        if (NEXT) {
            const float m_new = fmaxf(m_run, mx);
            if (__any(m_new > m_run)) {        // rescale only when some query's running max moved
                const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * scale_log2e);
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < 3; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
                m_run = m_new;
            }
        }
    };

    {
        const int nfull = nkt - 1;          // tiles that have a successor
        int kt = 0;
        for (; kt + 2 <= nfull; kt += 2) {
            step(sa, sb, kt, std::true_type{});
            step(sb, sa, kt + 1, std::true_type{});
        }
        if (kt < nfull) {
            step(sa, sb, kt, std::true_type{});
            step(sb, sa, kt + 1, std::false_type{});
        } else {
            step(sa, sb, kt, std::false_type{});
        }
    }
#undef AP_KRD
#undef AP_VTR
#undef AP_EXP
#undef AP_PV
#undef AP_MIX
#undef AP_PAIR
#undef AP_PFIN
#undef AP_SB
#undef AP_PV1
#undef AP_MX4

    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = 1.0f / l_tot;
    if (LSE && q_ok && h == 0) LSE[(int64_t)bh * Lq + qi] = m_run * scale_log2e + __builtin_amdgcn_logf(l_tot);  // log2 domain
    if (q_ok) {
        const int C = heads * 96;
        bf16_t* orow = O + ((int64_t)b * Lq + qi) * C + g * 96;
        const bf16_t* qrow = Qb + (int64_t)qi * 96;
#pragma unroll
        for (int db = 0; db < 3; ++db)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const int d = 32 * db + 8 * i4 + 4 * h;
                float4 v = make_float4(o[db][4 * i4 + 0] * inv, o[db][4 * i4 + 1] * inv, o[db][4 * i4 + 2] * inv,
                                       o[db][4 * i4 + 3] * inv);
                if (ADD_Q) {
                    const float4 qq = load4(qrow + d);
                    v.x += qq.x; v.y += qq.y; v.z += qq.z; v.w += qq.w;
                }
                store4(orow + d, v);
            }
    }
}

// ------------------------------------------------------------------------------------------------
// exact fp32 path: one query per thread, 32-key tiles in LDS (broadcast reads).
// ------------------------------------------------------------------------------------------------
#define F_KT 32
__global__ __launch_bounds__(128) void attn_fwd_f32_kernel(const float* __restrict__ Q, const float* __restrict__ Kt,
                                                           const float* __restrict__ V, float* __restrict__ O,
                                                           float* __restrict__ LSE, int heads, int Lq, int Lk, float scale,
                                                           int add_q) {
    __shared__ __attribute__((aligned(16))) float sK[F_KT * 96];
    __shared__ __attribute__((aligned(16))) float sV[F_KT * 96];
    const int bh = blockIdx.y;
    const int b = bh / heads, g = bh - b * heads;
    int qi = blockIdx.x * 128 + threadIdx.x;
    const bool q_ok = qi < Lq;
    qi = q_ok ? qi : Lq - 1;
    const float* qrow = Q + ((int64_t)bh * Lq + qi) * 96;
    float q[96], o[96];
#pragma unroll
    for (int d = 0; d < 96; d += 4) {
        const float4 v = load4(qrow + d);
        q[d] = v.x; q[d + 1] = v.y; q[d + 2] = v.z; q[d + 3] = v.w;
        o[d] = o[d + 1] = o[d + 2] = o[d + 3] = 0.f;
    }
    float m_run = -INFINITY, l_run = 0.f;
    const float* Kb = Kt + (int64_t)bh * Lk * 96;
    const float* Vb = V + (int64_t)bh * Lk * 96;
    for (int k0 = 0; k0 < Lk; k0 += F_KT) {
        __syncthreads();
        for (int i = threadIdx.x; i < F_KT * 24; i += 128) {
            const int row = i / 24, c4 = i - row * 24;
            float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
            if (k0 + row < Lk) {
                kv = load4(Kb + (int64_t)(k0 + row) * 96 + 4 * c4);
                vv = load4(Vb + (int64_t)(k0 + row) * 96 + 4 * c4);
            }
            *reinterpret_cast<float4*>(sK + row * 96 + 4 * c4) = kv;
            *reinterpret_cast<float4*>(sV + row * 96 + 4 * c4) = vv;
        }
        __syncthreads();
        const int nk = min(F_KT, Lk - k0);
        float sc[F_KT];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < F_KT; ++j) {
            float a = 0.f;
#pragma unroll
            for (int d = 0; d < 96; d += 4) {
                const float4 kv = *reinterpret_cast<const float4*>(sK + j * 96 + d);
                a = fmaf(q[d], kv.x, a); a = fmaf(q[d + 1], kv.y, a);
                a = fmaf(q[d + 2], kv.z, a); a = fmaf(q[d + 3], kv.w, a);
            }
            a = (j < nk) ? a * scale : -INFINITY;
            sc[j] = a;
            mx = fmaxf(mx, a);
        }
        const float m_new = fmaxf(m_run, mx);
        const float alpha = expf(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < 96; ++d) o[d] *= alpha;
#pragma unroll
        for (int j = 0; j < F_KT; ++j) {
            const float p = expf(sc[j] - m_new);
            l_run += p;
#pragma unroll
            for (int d = 0; d < 96; d += 4) {
                const float4 vv = *reinterpret_cast<const float4*>(sV + j * 96 + d);
                o[d] = fmaf(p, vv.x, o[d]); o[d + 1] = fmaf(p, vv.y, o[d + 1]);
                o[d + 2] = fmaf(p, vv.z, o[d + 2]); o[d + 3] = fmaf(p, vv.w, o[d + 3]);
            }
        }
    }
    if (q_ok) {
        const float inv = 1.0f / l_run;
        if (LSE) LSE[(int64_t)bh * Lq + qi] = (m_run + logf(l_run)) * 1.44269504088896340736f;   // log2 units
        float* orow = O + ((int64_t)b * Lq + qi) * (heads * 96) + g * 96;
#pragma unroll
        for (int d = 0; d < 96; d += 4) {
            float4 v = make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
            if (add_q) { v.x += q[d]; v.y += q[d + 1]; v.z += q[d + 2]; v.w += q[d + 3]; }
            store4(orow + d, v);
        }
    }
}

// attention_w64.hip
int attn_fwd_w64_prepare();
int attn_fwd_w64_launch(const void* q, const void* k, const void* v, void* out, float* lse, int B, int heads, int Lq, int Lk,
                        float scale_log2e, int add_q, hipStream_t st);

// True when the 16-bit forward of this shape runs in the 64-query kernel, whose scores (and saved lse) are those of the PRE-SCALED
// 16-bit queries round16(q * scale * log2e); the backward (attention_bwd.hip) recomputes its scores from the same values.
bool attn_fwd_prescales_q(int Lq, int Lk) {
    static const bool w64_env = !(getenv("MVIT_ATT_W64") && atoi(getenv("MVIT_ATT_W64")) == 0);
    return w64_env && Lk >= 64 && Lq >= 128;
}

// (round 4 built a key-split form of the ragged last query tile behind a second entry point, mvit_attention_fwd_ws: measured, not
// adopted, and taken out of the library in round 5 -- tools/probes/attn_fwd_keysplit.patch restores it)
extern "C" int mvit_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, int B, int heads,
                                  int Lq, int Lk, float scale, int add_q, int act_dtype, void* stream) {
    if (!q || !k || !v || !out || B <= 0 || heads <= 0 || Lq <= 0 || Lk <= 0) return MVIT_EINVAL;
    hipStream_t st = as_stream(stream);
    if ((int64_t)B * heads > 65535) return MVIT_EINVAL;
    if (act_dtype == MVIT_BF16) {
        // default: 64 queries per wave, one wave per SIMD (attention_w64.hip; +11 % on the model's shapes); MVIT_ATT_W64=0 selects the
        // 32-query kernels below, which also serve short sequences
        if (attn_fwd_prescales_q(Lq, Lk)) {
            static DevFlags wattr_done_tab; DevFlag wattr_done = dev_flag(wattr_done_tab);
            if (!wattr_done) { const int rc = attn_fwd_w64_prepare(); if (rc != MVIT_OK) return rc; wattr_done = true; }
            const int rc = attn_fwd_w64_launch(q, k, v, out, lse, B, heads, Lq, Lk, scale * 1.44269504088896340736f, add_q, st);
            if (rc != MVIT_OK) return rc;
            MVIT_LAUNCH_CHECK();
            return MVIT_OK;
        }
        static const bool pipe_env = !(getenv("MVIT_ATT_PIPE") && atoi(getenv("MVIT_ATT_PIPE")) == 0);   // default: software-pipelined kernel
        if (pipe_env) {
            dim3 grid((Lq + A_QB - 1) / A_QB, B * heads);
            const float sl2 = scale * 1.44269504088896340736f;
            static const bool slot_env = getenv("MVIT_ATT_SLOT") && atoi(getenv("MVIT_ATT_SLOT")) != 0;
            static DevFlags pattr_done_tab; DevFlag pattr_done = dev_flag(pattr_done_tab);
            if (!pattr_done) {
                if (hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_pipe_kernel<true, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 2 * AP_RING) != hipSuccess ||
                    hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_pipe_kernel<false, false>), hipFuncAttributeMaxDynamicSharedMemorySize, 2 * AP_RING) != hipSuccess ||
                    hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_pipe_kernel<true, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 2 * AP_RING) != hipSuccess ||
                    hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_pipe_kernel<false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 2 * AP_RING) != hipSuccess)
                    return MVIT_ELAUNCH;
                pattr_done = true;
            }
#define PIPE_LAUNCH(AQ, SL) hipLaunchKernelGGL((attn_fwd_pipe_kernel<AQ, SL>), grid, dim3(256), 2 * AP_RING, st, (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)out, lse, heads, Lq, Lk, sl2)
            if (slot_env) { if (add_q) PIPE_LAUNCH(true, true); else PIPE_LAUNCH(false, true); }
            else { if (add_q) PIPE_LAUNCH(true, false); else PIPE_LAUNCH(false, false); }
#undef PIPE_LAUNCH
            MVIT_LAUNCH_CHECK();
            return MVIT_OK;
        }
        static const int nw_env = getenv("MVIT_ATT_WAVES") ? atoi(getenv("MVIT_ATT_WAVES")) : 4;
        const int NWr = nw_env == 8 ? 8 : 4;
        dim3 grid((Lq + 32 * NWr - 1) / (32 * NWr), B * heads);
        const float sl2 = scale * 1.44269504088896340736f;
        static DevFlags attr_done_tab; DevFlag attr_done = dev_flag(attr_done_tab);
        if (!attr_done) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_bf16_kernel<true, 4>), hipFuncAttributeMaxDynamicSharedMemorySize, A_STAGES * A_TILEB) != hipSuccess ||
                hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_bf16_kernel<false, 4>), hipFuncAttributeMaxDynamicSharedMemorySize, A_STAGES * A_TILEB) != hipSuccess ||
                hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_bf16_kernel<true, 8>), hipFuncAttributeMaxDynamicSharedMemorySize, A_STAGES * A_TILEB) != hipSuccess ||
                hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_bf16_kernel<false, 8>), hipFuncAttributeMaxDynamicSharedMemorySize, A_STAGES * A_TILEB) != hipSuccess)
                return MVIT_ELAUNCH;
            attr_done = true;
        }
#define ATT_LAUNCH(AQ, NWW) hipLaunchKernelGGL((attn_fwd_bf16_kernel<AQ, NWW>), grid, dim3(64 * NWW), A_STAGES * A_TILEB, st, (const bf16_t*)q, \
                                               (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)out, lse, heads, Lq, Lk, sl2)
        if (add_q) { if (NWr == 8) ATT_LAUNCH(true, 8); else ATT_LAUNCH(true, 4); }
        else { if (NWr == 8) ATT_LAUNCH(false, 8); else ATT_LAUNCH(false, 4); }
#undef ATT_LAUNCH
    } else if (act_dtype == MVIT_F32) {
        dim3 grid((Lq + 127) / 128, B * heads);
        hipLaunchKernelGGL(attn_fwd_f32_kernel, grid, dim3(128), 0, st, (const float*)q, (const float*)k, (const float*)v,
                           (float*)out, lse, heads, Lq, Lk, scale, add_q);
    } else {
        return MVIT_EDTYPE;
    }
    MVIT_LAUNCH_CHECK();
    return MVIT_OK;
}
