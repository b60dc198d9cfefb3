// Causal softmax attention over packed sequences of different lengths, grouped heads, forward and backward.
//
//   o_i = sum_{j <= i + Lk - Lq} softmax_j(scale q_i . k_j) v_j          per sequence and head; key head = head / (Hq / Hkv)
//   dV = P^T dO,  dS = P o (dO V^T - rowsum(dO o O)),  dQ = scale dS K,  dK = scale dS^T Q
//
// One wave owns 32 query rows (forward, dQ) or 32 or 64 key rows (dK / dV); the 64-row tiles of the other side pass through LDS, double-buffered and written there by the
// loads themselves (tile t + 1 in flight under the products of tile t).  "Swapped" products: S^T = K Q^T puts one query into one
// lane's column, so that softmax is lane-local, and the accumulator layout of P^T is, up to a fixed order of the contraction index, the operand
// layout of the second product -- the transposed V / K / dO / Q fragments are read in that order by ds_read_b64_tr_b16, nothing is exchanged.
// The sequences' lengths live on the device only: seq_common.h maps slots to (sequence, tile).
//
// Bound by the matrix cores on long sequences: 16384 rows, 8 heads of width 64, forward 306 us = 898 TFLOP/s of the products it needs; 4 x 4096 rows, 16 heads of width 128 over 4
// key heads: forward 295 us = 931, dQ 386 us = 1069, dK / dV 540 us + 26 us for the parts' sums = 971 TFLOP/s of the products they do (bf16 library products of 8192^3 and
// more reach 1340 here).  On short ones by the chain of a sequence's tiles (7 ragged sequences of up to 2048 rows: 27, 29 and 40 + 7 us against 21 us of products in all), and under
// 256 rows by the launch.  (Medians of kernel traces in a steady run on cold inputs, scripts/sequence_kernels.py; single passes from idle clocks take up to a sixth longer.)
#include "packed_common.h"

// ------------------------------------------------------------------------------------------------------------------------------
// A block of the forward and dQ kernels: 128 query rows, 4 row groups of 32 x NG key groups of waves.  With two key groups alternate 64-key tiles pass through LDS two
// per step and the groups join their sums at the end: a causal tile's time is a chain of (its keys / 64 NG) dependent steps, and with few sequences the
// longest chain, not the chip, is what a launch waits for.
// ------------------------------------------------------------------------------------------------------------------------------
struct PackedRows {
    SeqSlot s;
    PackedBlock blk;
    int kstart, klen, shift, q0, qi, nstep, w_end, grp, rw;
};
template <int RW, int NG>
__device__ __forceinline__ bool packed_rows(const PackedArgs& a, PackedRows& r, bf16_t* out) {
    constexpr int BM = 32 * RW;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    r.grp = wave / RW;
    r.rw = wave % RW;
    r.blk = packed_block(a, a.hq);
    r.s = seq_find_longest<BM, false>(a.cu_q, a.nseq, a.rows_q, r.blk.slot, a.nslots);
    if (r.s.tile < 0 || r.s.tile * BM >= r.s.len) return false;
    if (r.s.seq == a.nseq) {
        packed_zero_rows<BM, 64 * RW * NG>(out, a.hq, a.dim, r.s, r.blk.head);
        return false;
    }
    r.kstart = seq_cu(a.cu_k, r.s.seq, a.rows_k);
    r.klen = max(0, seq_cu(a.cu_k, r.s.seq + 1, a.rows_k) - r.kstart);
    r.shift = r.klen - r.s.len;                                                 // query i sees keys 0 .. i + shift
    r.q0 = r.s.tile * BM + r.rw * 32;
    r.qi = r.q0 + (lane & 31);
    const int k_end = min(r.klen, min(r.s.tile * BM + BM, r.s.len) + r.shift);     // of the block (<= 0: nothing to see)
    r.w_end = min(r.klen, min(r.q0 + 32, r.s.len) + r.shift);                   // of this wave
    r.nstep = (max(k_end, 0) + 64 * NG - 1) / (64 * NG);
    return true;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Forward.  Online softmax in the exp2 domain with fp32 maximum, sum and accumulator; P is rounded to bf16 (at most 2^-8 of a weight, the precision
// of V itself) because the second product runs on the matrix cores; REST adds a product with what that left over.  The running maximum is "sum-triggered": a tile is exponentiated against the
// maximum as it stands, and only a lane whose partial row sum passes 2^8 (inf and NaN too) has the tile redone with its exact maximum -- no
// per-tile maximum tree in the steady state.  A wave's first tile always takes its maximum; a row that sees nothing of it (the second key group's first tile may lie
// behind it) sees nothing after it either.
// ------------------------------------------------------------------------------------------------------------------------------
template <int DH, int RW, int NG, int WPE, bool REST>
__global__ void __launch_bounds__(64 * RW * NG, WPE) packed_fwd_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    PackedRows r;
    if (!packed_rows<RW, NG>(a, r, a.out)) return;
    bf16x8_t qf[G::KS];
    packed_row_frags<DH>(qf, a.q + (int64_t)(r.s.start + r.qi) * a.q_row + r.blk.head * a.q_head, r.qi < r.s.len, a.dim);
    f32x16_t oacc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) oacc[d] = packed_splat(0.f);
    float m_run = -INFINITY, mc = 0.f, l_run = 0.f;                             // mc: m_run in the exp2 domain, 0 while there is none; l_run: this lane's half
    const float c2 = a.scale * 1.4426950408889634f;

    const bf16_t* kp = a.k + (int64_t)r.kstart * a.k_row + r.blk.kvh * a.k_head;
    const bf16_t* vp = a.v + (int64_t)r.kstart * a.v_row + r.blk.kvh * a.v_head;
    const int64_t k_step = 64 * NG * a.k_row, v_step = 64 * NG * a.v_row;
    PackedDma<DH, RW * NG, NG, (DH <= 64)> st;
    st.init(wave, lane, a.dim, a.k_row, a.v_row);
    auto load = [&](int t) {                                                    // (called for t = 0, 1, 2 ..)
        char* to = smem + (t & 1) * 2 * NG * G::TILE;
        st.load(wave, kp, seq_bytes_left(r.klen - t * 64 * NG, a.k_row * 2, a.dim), to, vp, seq_bytes_left(r.klen - t * 64 * NG, a.v_row * 2, a.dim), to + NG * G::TILE);
        kp += k_step;
        vp += v_step;
    };
    PackedLane<DH> at;
    at.init(lane);

    if (r.nstep > 0) load(0);
    for (int t = 0; t < r.nstep; ++t) {
        const char* kt_ = smem + (t & 1) * 2 * NG * G::TILE + r.grp * G::TILE;
        const char* vt_ = kt_ + NG * G::TILE;
        st.land();
        __syncthreads();
        if (t + 1 < r.nstep) load(t + 1);
        const int k0 = (t * NG + r.grp) * 64;
        if (k0 >= r.w_end) continue;                                            // (wave-uniform) nothing of this tile is visible to these 32 rows
        at.forget();
        bool with_max = t == 0;
        bf16x8_t pf[4], pr[REST ? 4 : 1];
        float psum;
        for (;;) {
            f32x16_t sacc[2] = {packed_splat(0.f), packed_splat(0.f)};
            bf16x8_t kf[2][G::KS];                                              // all of the tile's fragments requested before the first product
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) kf[kt][ks] = at.row_frag(kt_ + kt * 32 * G::PITCH, ks);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sacc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kt][ks], qf[ks], sacc[kt], 0, 0, 0);
            if (k0 + 64 > r.klen || k0 + 63 > r.q0 + r.shift) {                 // the tile crosses the last key or the diagonal of these rows
                int lim = min(r.klen, r.qi + r.shift + 1) - k0 - 4 * h;
                asm volatile("" : "+v"(lim));                                   // (the comparisons stay in this branch)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sacc[kt][e] = kt * 32 + seq_crow(e) < lim ? sacc[kt][e] : -INFINITY;
            }
            if (with_max) {
                float tm = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) tm = fmaxf(tm, sacc[kt][e]);
                const float m_new = fmaxf(m_run, seq_xmax32(tm));
                const float mc_new = m_new == -INFINITY ? 0.f : m_new * c2;
                const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - mc_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < G::DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[d][e] *= alpha;
                m_run = m_new;
                mc = mc_new;
            }
            float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[kt][8 * s2 + e], c2, -mc));
                        ps[e & 3] += p[e];
                    }
                    pf[2 * kt + s2] = seq_pack8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
                    if (REST) pr[REST ? 2 * kt + s2 : 0] = seq_rest8(p, pf[2 * kt + s2]);
                }
            psum = (ps[0] + ps[1]) + (ps[2] + ps[3]);
            if (with_max || __builtin_amdgcn_ballot_w64(!(psum <= 256.f)) == 0) break;
            with_max = true;
        }
        l_run += psum;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < G::DT; ++d) {
                const bf16x8_t vf = at.tr_frag(vt_ + ks * 16 * G::PITCH, d);
                if (REST) oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pr[REST ? ks : 0], oacc[d], 0, 0, 0);
                oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[ks], oacc[d], 0, 0, 0);
            }
    }
    float l = 0.f;
    if constexpr (NG == 1) {
        l = seq_xsum32(l_run);
    } else {
        // the second key group's sums join the first's: through LDS, register by register (lane = the same row and columns in both)
        __syncthreads();
        float* xs = reinterpret_cast<float*>(smem) + r.rw * (G::DT * 16 + 2) * 64 + lane;
        if (r.grp == 1) {
            xs[0] = m_run == -INFINITY ? -INFINITY : mc;
            xs[64] = l_run;
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) xs[(2 + d * 16 + e) * 64] = oacc[d][e];
        }
        __syncthreads();
        if (r.grp == 0) {
            const float m1 = xs[0], m0 = m_run == -INFINITY ? -INFINITY : mc, mx = fmaxf(m0, m1), l1 = xs[64];
            // (a part without a maximum has nothing, or NaN: it goes in as it is)
            const float f0 = m0 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m0 - mx), f1 = m1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m1 - mx);
            mc = mx == -INFINITY ? 0.f : mx;
            l = seq_xsum32(l_run * f0 + l1 * f1);
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[d][e] = oacc[d][e] * f0 + xs[(2 + d * 16 + e) * 64] * f1;
        }
    }
    if (r.grp == 0 && a.lse && h == 0 && r.qi < r.s.len)
        a.lse[(int64_t)r.blk.head * a.rows_q + r.s.start + r.qi] = l == 0.f ? -INFINITY : mc * 0.6931471805599453f + __logf(l);
    __syncthreads();                                                            // tiles and exchange area become the waves' output regions
    if (r.grp == 0 && r.q0 < r.s.len) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t to = ((int64_t)(r.s.start + r.q0) * a.hq + r.blk.head) * a.dim;
        packed_write_rows<DH>(smem + r.rw * 32 * G::PITCH, oacc, inv, a.out + to, (int64_t)a.hq * a.dim, min(32, r.s.len - r.q0), a.dim);
        if (a.out_lo) {
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[d][e] = oacc[d][e] * inv - bf16_to_f32(f32_to_bf16(oacc[d][e] * inv));
            packed_write_rows<DH>(smem + r.rw * 32 * G::PITCH, oacc, 1.f, a.out_lo + to, (int64_t)a.hq * a.dim, min(32, r.s.len - r.q0), a.dim);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// Backward, dQ: the forward's walk over the keys with P recomputed from the log-sum-exp.  delta = rowsum(dO o O) of the wave's rows is formed from the
// operand fragments, written out for the other kernel, and fed negated as the accumulator INPUT of dP^T = V dO^T, so that dS = P o (dP - delta) costs
// no subtraction.  dS is rounded to bf16 for the last product (REST: and what that left over), like P in the forward.  delta takes O with the 16 bits that its rounding left over: where a row sees few
// keys, dP - delta is a small difference, and the rounding of O alone would be as large an error in it as that of dS (a 5720-row batch: dQ 0.0026 off in
// norm with it, 0.0024 without; sequences of a few tokens 0.0035 and 0.0024).
// ------------------------------------------------------------------------------------------------------------------------------
template <int DH, int RW, int NG, int WPE, bool REST>
__global__ void __launch_bounds__(64 * RW * NG, WPE) packed_dq_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    PackedRows r;
    if (!packed_rows<RW, NG>(a, r, a.dq)) return;
    bf16x8_t qf[G::KS], gf[G::KS];
    const int64_t qrow = r.s.start + r.qi;
    packed_row_frags<DH>(qf, a.q + qrow * a.q_row + r.blk.head * a.q_head, r.qi < r.s.len, a.dim);
    packed_row_frags<DH>(gf, a.dout + qrow * a.g_row + r.blk.head * a.g_head, r.qi < r.s.len, a.dim);
    float delta = 0.f, lse2 = INFINITY;                                         // a row that sees nothing, or none at all: exp2(x - inf) = 0
    {
        bf16x8_t of[G::KS], ol[G::KS];
        packed_row_frags<DH>(of, a.o + (qrow * a.hq + r.blk.head) * a.dim, r.qi < r.s.len, a.dim);
        packed_row_frags<DH>(ol, a.out_lo + (qrow * a.hq + r.blk.head) * a.dim, r.qi < r.s.len, a.dim);
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                delta = __builtin_fmaf(bf16_to_f32((bf16_t)gf[ks][e]), bf16_to_f32((bf16_t)of[ks][e]) + bf16_to_f32((bf16_t)ol[ks][e]), delta);
        delta = seq_xsum32(delta);
        if (r.qi < r.s.len) {
            const float lse = a.lse[(int64_t)r.blk.head * a.rows_q + qrow];
            lse2 = lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
            if (h == 0 && r.grp == 0) a.delta[(int64_t)r.blk.head * a.rows_q + qrow] = delta;
        }
    }
    f32x16_t acc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) acc[d] = packed_splat(0.f);
    const float c2 = a.scale * 1.4426950408889634f;
    const bf16_t* kp = a.k + (int64_t)r.kstart * a.k_row + r.blk.kvh * a.k_head;
    const bf16_t* vp = a.v + (int64_t)r.kstart * a.v_row + r.blk.kvh * a.v_head;
    const int64_t k_step = 64 * NG * a.k_row, v_step = 64 * NG * a.v_row;
    PackedDma<DH, RW * NG, NG, (DH <= 64)> st;
    st.init(wave, lane, a.dim, a.k_row, a.v_row);
    auto load = [&](int t) {                                                    // (called for t = 0, 1, 2 ..)
        char* to = smem + (t & 1) * 2 * NG * G::TILE;
        st.load(wave, kp, seq_bytes_left(r.klen - t * 64 * NG, a.k_row * 2, a.dim), to, vp, seq_bytes_left(r.klen - t * 64 * NG, a.v_row * 2, a.dim), to + NG * G::TILE);
        kp += k_step;
        vp += v_step;
    };
    PackedLane<DH> at;
    at.init(lane);

    if (r.nstep > 0) load(0);
    for (int t = 0; t < r.nstep; ++t) {
        const char* kt_ = smem + (t & 1) * 2 * NG * G::TILE + r.grp * G::TILE;
        const char* vt_ = kt_ + NG * G::TILE;
        st.land();
        __syncthreads();
        if (t + 1 < r.nstep) load(t + 1);
        const int k0 = (t * NG + r.grp) * 64;
        if (k0 >= r.w_end) continue;
        at.forget();
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            f32x16_t sacc = packed_splat(0.f), dp = packed_splat(-delta);
            bf16x8_t ka[G::KS], va[G::KS];                                      // (a product's fragments are requested one product ahead: 4 x 4096 rows 397 us, else 408)
            ka[0] = at.row_frag(kt_ + kt * 32 * G::PITCH, 0);
            va[0] = at.row_frag(vt_ + kt * 32 * G::PITCH, 0);
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                if (ks + 1 < G::KS) {
                    ka[ks + 1] = at.row_frag(kt_ + kt * 32 * G::PITCH, ks + 1);
                    va[ks + 1] = at.row_frag(vt_ + kt * 32 * G::PITCH, ks + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[ks], qf[ks], sacc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[ks], gf[ks], dp, 0, 0, 0);
            }
            if (k0 + 64 > r.klen || k0 + 63 > r.q0 + r.shift) {
                int lim = min(r.klen, r.qi + r.shift + 1) - k0 - 32 * kt - 4 * h;
                asm volatile("" : "+v"(lim));
#pragma unroll
                for (int e = 0; e < 16; ++e) sacc[e] = seq_crow(e) < lim ? sacc[e] : -INFINITY;
            }
            bf16x8_t ds[2], dr[REST ? 2 : 1];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[8 * s2 + e], c2, -lse2)) * dp[8 * s2 + e];
                ds[s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
                if (REST) dr[REST ? s2 : 0] = seq_rest8(x, ds[s2]);
            }
            bf16x8_t kfr[2 * G::DT];
            kfr[0] = at.tr_frag(kt_ + kt * 32 * G::PITCH, 0);
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < G::DT; ++d) {
                    const int n = s2 * G::DT + d;
                    if (n + 1 < 2 * G::DT) kfr[n + 1] = at.tr_frag(kt_ + (kt * 2 + (n + 1) / G::DT) * 16 * G::PITCH, (n + 1) % G::DT);
                    __builtin_amdgcn_sched_barrier(0);
                    const bf16x8_t kf = kfr[n];
                    if (REST) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, dr[REST ? s2 : 0], acc[d], 0, 0, 0);
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, ds[s2], acc[d], 0, 0, 0);
                }
        }
    }
    if constexpr (NG == 2) {
        __syncthreads();
        float* xs = reinterpret_cast<float*>(smem) + r.rw * G::DT * 16 * 64 + lane;
        if (r.grp == 1)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) xs[(d * 16 + e) * 64] = acc[d][e];
        __syncthreads();
        if (r.grp == 0)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][e] += xs[(d * 16 + e) * 64];
    }
    __syncthreads();
    if (r.grp == 0 && r.q0 < r.s.len)
        packed_write_rows<DH>(smem + r.rw * 32 * G::PITCH, acc, a.scale, a.dq + ((int64_t)(r.s.start + r.q0) * a.hq + r.blk.head) * a.dim, (int64_t)a.hq * a.dim,
                              min(32, r.s.len - r.q0), a.dim);
}

// ------------------------------------------------------------------------------------------------------------------------------
// C entry points
// ------------------------------------------------------------------------------------------------------------------------------
static int packed_check(const char* what, const PackedArgs& a) {
    GENIE_CHECK_ARG(a.q && a.k && a.v && a.cu_q && a.cu_k, "%s: null pointer", what);
    GENIE_CHECK_ARG(a.nseq >= 0 && a.rows_q >= 0 && a.rows_k >= 0 && a.rows_q <= (1 << 30) && a.rows_k <= (1 << 30), "%s: bad sizes", what);
    GENIE_CHECK_ARG(a.hkv > 0 && a.hq > 0 && a.hq % a.hkv == 0, "%s: %d query heads are no multiple of %d key heads", what, a.hq, a.hkv);
    GENIE_CHECK_ARG(a.dim > 0 && a.dim % 8 == 0 && a.dim <= 128, "%s: head width %d (a multiple of 8 up to 128 is supported)", what, a.dim);
    GENIE_CHECK_ARG(a.scale > 0.f && a.scale < 1e30f, "%s: scale must be positive and finite", what);
    const int64_t s[8] = {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.g_row, a.g_head};
    for (int i = 0; i < 8; ++i) GENIE_CHECK_ARG(s[i] >= 0 && s[i] % 8 == 0, "%s: strides must be multiples of 8 elements", what);
    for (int i = 0; i < 8; i += 2)
        GENIE_CHECK_ARG(s[i] >= a.dim && s[i] < (1 << 21), "%s: row stride %lld (the head width up to 2^21 elements is supported)", what, (long long)s[i]);
    return GENIE_OK;
}

// Two key groups per block (half the chain of steps, but waves without work where a sequence has only a tile or two, and at head widths above 64 one coupled block per CU
// instead of two independent ones) from an average of 512 rows per sequence on, and while the launch leaves CUs short of blocks.  Measured one / two groups, us,
// 16 query heads over 4 key heads: forward at width 64, one sequence of 1024 / 4096 / 8192: 18.2 / 15.3, 61.5 / 52.3, 158.0 / 157.3, at 40 x 100 rows 11.2 / 16.1;
// width 128: 28.2 / 22.6, 101.2 / 91.2, 292.7 / 290.5, 4 x 2048: 89.0 / 97.8.  Backward at width 64: 52.1 / 49.3, 174.5 / 162.3, 504 / 520.
// At widths up to 64 these blocks hold 64 rows instead of 128 while there are few of them: forward, 128 / 64 rows, 8 heads, one sequence of 1024 / 4096 / 8192:
// 15.1 / 12.4, 43.2 / 38.6, 94.4 / 99.9; 5720 ragged rows 30.6 / 26.6 (dQ 33.2 / 30.5); 4 x 2048 31.0 / 34.7.
static bool packed_two_groups(const PackedArgs& a, int64_t most) { return a.rows_q >= 512ll * a.nseq && packed_few(a.rows_q, a.hq, most); }

template <int DH, int RW, int NG, int WPE, bool REST>
static int packed_fwd_run(PackedArgs& a, void* stream) {
    a.nslots = a.rows_q / (32 * RW) + a.nseq + 1;
    return packed_launch(packed_fwd_kernel<DH, RW, NG, WPE, REST>, a, (int64_t)a.nslots * a.hq, 64 * RW * NG, 4 * NG * PackedGeo<DH>::TILE, stream);
}
template <int DH, int RW, int NG, int WPE, bool REST>
static int packed_dq_run(PackedArgs& a, void* stream) {
    a.nslots = a.rows_q / (32 * RW) + a.nseq + 1;
    return packed_launch(packed_dq_kernel<DH, RW, NG, WPE, REST>, a, (int64_t)a.nslots * a.hq, 64 * RW * NG, 4 * NG * PackedGeo<DH>::TILE, stream);
}

template <int DH>
static int packed_fwd_dispatch(PackedArgs& a, void* stream) {
    if (packed_exact(a)) return packed_fwd_run<DH, 4, 1, 1, true>(a, stream);
    if (DH <= 64 && packed_two_groups(a, 448)) return packed_fwd_run<DH <= 64 ? DH : 64, 2, 2, 2, false>(a, stream);
    if (packed_two_groups(a, DH <= 64 ? (1ll << 31) : 512)) return packed_fwd_run<DH, 4, 2, DH <= 64 ? 4 : 2, false>(a, stream);
    return packed_fwd_run<DH, 4, 1, DH <= 64 ? 3 : 2, false>(a, stream);
}

template <int DH>
static int packed_bwd_dispatch(PackedArgs& a, void* stream) {
    int rc;
    if (packed_exact(a)) rc = packed_dq_run<DH, 4, 1, 1, true>(a, stream);
    else if (DH <= 64 && packed_two_groups(a, 448)) rc = packed_dq_run<DH <= 64 ? DH : 64, 2, 2, 2, false>(a, stream);
    else if (packed_two_groups(a, 512)) rc = packed_dq_run<DH, 4, 2, 2, false>(a, stream);
    else rc = packed_dq_run<DH, 4, 1, DH <= 64 ? 3 : 2, false>(a, stream);
    return rc != GENIE_OK ? rc : packed_dkv_run(a, stream);
}

extern "C" int genie_packed_attention_fwd(const void* q, const void* k, const void* v, void* out, void* out_lo, float* lse, const int32_t* cu_q, const int32_t* cu_k, int nseq,
                                          int rows_q, int rows_k, int hq, int hkv, int dim, const int64_t* q_strides, const int64_t* k_strides,
                                          const int64_t* v_strides, float scale, void* stream) {
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides, "genie_packed_attention_fwd: null strides");
    PackedArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.out = (bf16_t*)out; a.out_lo = (bf16_t*)out_lo; a.lse = lse;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseq = nseq; a.rows_q = rows_q; a.rows_k = rows_k; a.hq = hq; a.hkv = hkv; a.dim = dim; a.scale = scale;
    a.q_row = q_strides[0]; a.q_head = q_strides[1]; a.k_row = k_strides[0]; a.k_head = k_strides[1]; a.v_row = v_strides[0]; a.v_head = v_strides[1];
    a.g_row = a.q_row; a.g_head = a.q_head;
    const int rc = packed_check("genie_packed_attention_fwd", a);
    if (rc != GENIE_OK) return rc;
    GENIE_CHECK_ARG(out != nullptr, "genie_packed_attention_fwd: null pointer");
    if (rows_q == 0) return GENIE_OK;
    if (dim <= 32) return packed_fwd_dispatch<32>(a, stream);
    if (dim <= 64) return packed_fwd_dispatch<64>(a, stream);
    if (dim <= 96) return packed_fwd_dispatch<96>(a, stream);
    return packed_fwd_dispatch<128>(a, stream);
}

extern "C" int genie_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_lo, const void* dout, const float* lse, float* ws, int64_t ws_floats, void* dq,
                                          void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, int nseq, int rows_q, int rows_k, int hq, int hkv, int dim,
                                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* dout_strides, float scale,
                                          void* stream) {
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides && dout_strides, "genie_packed_attention_bwd: null strides");
    PackedArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.o = (const bf16_t*)out; a.out_lo = (bf16_t*)const_cast<void*>(out_lo); a.dout = (const bf16_t*)dout;
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.lse = const_cast<float*>(lse); a.delta = ws;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseq = nseq; a.rows_q = rows_q; a.rows_k = rows_k; a.hq = hq; a.hkv = hkv; a.dim = dim; a.scale = scale;
    a.q_row = q_strides[0]; a.q_head = q_strides[1]; a.k_row = k_strides[0]; a.k_head = k_strides[1]; a.v_row = v_strides[0]; a.v_head = v_strides[1];
    a.g_row = dout_strides[0]; a.g_head = dout_strides[1];
    const int rc = packed_check("genie_packed_attention_bwd", a);
    if (rc != GENIE_OK) return rc;
    GENIE_CHECK_ARG(out && out_lo && dout && lse && ws && dq && dk && dv, "genie_packed_attention_bwd: null pointer");
    GENIE_CHECK_ARG(ws_floats >= genie_packed_attention_bwd_ws_floats(nseq, rows_q, rows_k, hq, hkv, dim) && (uintptr_t)ws % 16 == 0,
                    "genie_packed_attention_bwd: workspace too small or not 16-byte aligned");
    if (dim <= 32) return packed_bwd_dispatch<32>(a, stream);
    if (dim <= 64) return packed_bwd_dispatch<64>(a, stream);
    if (dim <= 96) return packed_bwd_dispatch<96>(a, stream);
    return packed_bwd_dispatch<128>(a, stream);
}
