// Causal softmax attention over packed sequences of different lengths, grouped heads, forward and backward.
//
//   o_i = sum_{j <= i + Lk - Lq} softmax_j(scale q_i . k_j) v_j          per sequence and head; key head = head / (Hq / Hkv)
//   dV = P^T dO,  dS = P o (dO V^T - rowsum(dO o O)),  dQ = scale dS K,  dK = scale dS^T Q
//
// One wave owns 32 query rows (forward, dQ) or 32 key rows (dK / dV); the 64-row tiles of the other side pass through LDS, double-buffered, staged
// through registers (global load of tile t + 1 in flight under the products of tile t).  "Swapped" products: S^T = K Q^T puts one query into one
// lane's column, so that softmax is lane-local, and the accumulator layout of P^T is, up to a fixed order of the contraction index, the operand
// layout of the second product -- the transposed V / K / dO / Q fragments are read in that order by ds_read_b64_tr_b16, nothing is exchanged.
// The sequences' lengths live on the device only: seq_common.h maps slots to (sequence, tile).
#include "packed_common.h"

// ------------------------------------------------------------------------------------------------------------------------------
// Forward.  Online softmax in the exp2 domain with fp32 maximum, sum and accumulator; P is rounded to bf16 (at most 2^-8 of a weight, the precision
// of V itself) because the second product runs on the matrix cores.  The running maximum is "sum-triggered": a tile is exponentiated against the
// maximum as it stands, and only a lane whose partial row sum passes 2^8 (inf and NaN too) has the tile redone with its exact maximum -- no
// per-tile maximum tree in the steady state.  The first tile always takes its maximum, and every row that sees any key sees key 0.
// ------------------------------------------------------------------------------------------------------------------------------
#ifndef FWD_WPE
#define FWD_WPE 3
#endif
#ifdef FWD_DMA
#define FwdTiles PackedDma
#else
#define FwdTiles PackedTiles
#endif
template <int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? FWD_WPE : 2) packed_fwd_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    constexpr int BM = 32 * NW, NT = 64 * NW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const PackedBlock blk = packed_block(a, a.hq);
    const SeqSlot s = seq_find_longest<BM, false>(a.cu_q, a.nseq, a.rows_q, blk.slot, a.nslots);
    if (s.tile < 0 || s.tile * BM >= s.len) return;
    if (s.seq == a.nseq) {
        packed_zero_rows<BM, NT>(a.out, a.hq, a.dim, s, blk.head);
        return;
    }
    const int kstart = seq_cu(a.cu_k, s.seq, a.rows_k), klen = max(0, seq_cu(a.cu_k, s.seq + 1, a.rows_k) - kstart);
    const int shift = klen - s.len;                                             // query i sees keys 0 .. i + shift
    const int q0 = s.tile * BM + wave * 32, qi = q0 + (lane & 31);
    const int k_end = min(klen, min(s.tile * BM + BM, s.len) + shift);          // of the block (<= 0: nothing to see)
    const int w_end = min(klen, min(q0 + 32, s.len) + shift);                   // of this wave
    const int ntile = (max(k_end, 0) + 63) >> 6;

    bf16x8_t qf[G::KS];
    packed_row_frags<DH>(qf, a.q + (int64_t)(s.start + qi) * a.q_row + blk.head * a.q_head, qi < s.len, a.dim);
    f32x16_t oacc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) oacc[d] = packed_splat(0.f);
    float m_run = -INFINITY, mc = 0.f, l_run = 0.f;                             // mc: m_run in the exp2 domain, 0 while there is none; l_run: this lane's half
    const float c2 = a.scale * 1.4426950408889634f;

    const bf16_t* kp = a.k + (int64_t)kstart * a.k_row + blk.kvh * a.k_head;
    const bf16_t* vp = a.v + (int64_t)kstart * a.v_row + blk.kvh * a.v_head;
    FwdTiles<DH, NW> st;
    st.init(wave, lane, a.dim, a.k_row, a.v_row);
    const int64_t k_step = 64 * a.k_row, v_step = 64 * a.v_row;
    auto load = [&](int t) {                                                    // (called for t = 0, 1, 2 ..)
        char* to = smem + (t & 1) * 2 * G::TILE;
        st.load(wave, kp, seq_bytes_left(klen - t * 64, a.k_row * 2, a.dim), to, vp, seq_bytes_left(klen - t * 64, a.v_row * 2, a.dim), to + G::TILE);
        kp += k_step;
        vp += v_step;
    };
    PackedLane<DH> at;
    at.init(lane);

    if (ntile > 0) load(0);
    for (int t = 0; t < ntile; ++t) {
        char* kt_ = smem + (t & 1) * 2 * G::TILE;
        char* vt_ = kt_ + G::TILE;
        st.land(kt_, vt_);
        __syncthreads();
        if (t + 1 < ntile) load(t + 1);
        const int k0 = t * 64;
        if (k0 >= w_end) continue;                                              // (wave-uniform) nothing of this tile is visible to these 32 rows
        at.forget();
        bool with_max = t == 0;
        bf16x8_t pf[4];
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
            if (k0 + 64 > klen || k0 + 63 > q0 + shift) {                       // the tile crosses the last key or the diagonal of these rows
                int lim = min(klen, qi + shift + 1) - k0 - 4 * h;
                asm volatile("" : "+v"(lim));                                   // (the comparisons stay in this branch)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sacc[kt][r] = kt * 32 + seq_crow(r) < lim ? sacc[kt][r] : -INFINITY;
            }
            if (with_max) {
                float tm = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) tm = fmaxf(tm, sacc[kt][r]);
                const float m_new = fmaxf(m_run, seq_xmax32(tm));
                const float mc_new = m_new == -INFINITY ? 0.f : m_new * c2;
                const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - mc_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < G::DT; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[d][r] *= alpha;
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
                }
            psum = (ps[0] + ps[1]) + (ps[2] + ps[3]);
            if (with_max || __builtin_amdgcn_ballot_w64(!(psum <= 256.f)) == 0) break;
            with_max = true;
        }
        l_run += psum;
#ifdef FWD_ASM
        if constexpr (G::DT % 2 == 0) {
            const uint32_t vb = attn_lds_offset(vt_);
#pragma unroll
            for (int dd = 0; dd < G::DT; dd += 2) {
                const uint32_t a0 = vb + (at.tr0 ^ (dd * 64)), a1 = vb + (at.tr1 ^ (dd * 64)), a2 = vb + (at.tr0 ^ (dd * 64 + 64)), a3 = vb + (at.tr1 ^ (dd * 64 + 64));
                bf16x8_t f[4];
                seq_tr16x4<0, 16 * G::PITCH>(f, a0, a1, a2, a3);
                oacc[dd] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[0], pf[0], oacc[dd], 0, 0, 0);
                oacc[dd + 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[1], pf[0], oacc[dd + 1], 0, 0, 0);
                oacc[dd] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[2], pf[1], oacc[dd], 0, 0, 0);
                oacc[dd + 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[3], pf[1], oacc[dd + 1], 0, 0, 0);
                seq_tr16x4<32 * G::PITCH, 48 * G::PITCH>(f, a0, a1, a2, a3);
                oacc[dd] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[0], pf[2], oacc[dd], 0, 0, 0);
                oacc[dd + 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[1], pf[2], oacc[dd + 1], 0, 0, 0);
                oacc[dd] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[2], pf[3], oacc[dd], 0, 0, 0);
                oacc[dd + 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[3], pf[3], oacc[dd + 1], 0, 0, 0);
            }
        } else
#endif
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
                oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.tr_frag(vt_ + ks * 16 * G::PITCH, d), pf[ks], oacc[d], 0, 0, 0);
    }
    const float l = seq_xsum32(l_run);
    if (a.lse && h == 0 && qi < s.len)
        a.lse[(int64_t)blk.head * a.rows_q + s.start + qi] = l == 0.f ? -INFINITY : mc * 0.6931471805599453f + __logf(l);
    __syncthreads();                                                            // the staging tiles become the waves' output regions
    if (q0 < s.len)
        packed_write_rows<DH>(smem + wave * 32 * G::PITCH, oacc, l == 0.f ? 0.f : 1.f / l, a.out + ((int64_t)(s.start + q0) * a.hq + blk.head) * a.dim,
                              (int64_t)a.hq * a.dim, min(32, s.len - q0), a.dim);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Backward, dQ: the forward's walk over the keys with P recomputed from the log-sum-exp.  delta = rowsum(dO o O) of the wave's rows is formed from the
// operand fragments, written out for the other kernel, and fed negated as the accumulator INPUT of dP^T = V dO^T, so that dS = P o (dP - delta) costs
// no subtraction.  dS is rounded to bf16 for the last product, like P in the forward.
// ------------------------------------------------------------------------------------------------------------------------------
template <int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? 3 : 2) packed_dq_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    constexpr int BM = 32 * NW, NT = 64 * NW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const PackedBlock blk = packed_block(a, a.hq);
    const SeqSlot s = seq_find_longest<BM, false>(a.cu_q, a.nseq, a.rows_q, blk.slot, a.nslots);
    if (s.tile < 0 || s.tile * BM >= s.len) return;
    if (s.seq == a.nseq) {
        packed_zero_rows<BM, NT>(a.dq, a.hq, a.dim, s, blk.head);
        return;
    }
    const int kstart = seq_cu(a.cu_k, s.seq, a.rows_k), klen = max(0, seq_cu(a.cu_k, s.seq + 1, a.rows_k) - kstart);
    const int shift = klen - s.len;
    const int q0 = s.tile * BM + wave * 32, qi = q0 + (lane & 31);
    const int k_end = min(klen, min(s.tile * BM + BM, s.len) + shift), w_end = min(klen, min(q0 + 32, s.len) + shift);
    const int ntile = (max(k_end, 0) + 63) >> 6;

    bf16x8_t qf[G::KS], gf[G::KS];
    const int64_t qrow = s.start + qi;
    packed_row_frags<DH>(qf, a.q + qrow * a.q_row + blk.head * a.q_head, qi < s.len, a.dim);
    packed_row_frags<DH>(gf, a.dout + qrow * a.g_row + blk.head * a.g_head, qi < s.len, a.dim);
    float delta = 0.f, lse2 = INFINITY;                                         // a row that sees nothing, or none at all: exp2(x - inf) = 0
    {
        bf16x8_t of[G::KS];
        packed_row_frags<DH>(of, a.o + (qrow * a.hq + blk.head) * a.dim, qi < s.len, a.dim);
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(bf16_to_f32((bf16_t)gf[ks][e]), bf16_to_f32((bf16_t)of[ks][e]), delta);
        delta = seq_xsum32(delta);
        if (qi < s.len) {
            const float lse = a.lse[(int64_t)blk.head * a.rows_q + qrow];
            lse2 = lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
            if (h == 0) a.delta[(int64_t)blk.head * a.rows_q + qrow] = delta;
        }
    }
    f32x16_t acc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) acc[d] = packed_splat(0.f);
    const float c2 = a.scale * 1.4426950408889634f;
    const bf16_t* kp = a.k + (int64_t)kstart * a.k_row + blk.kvh * a.k_head;
    const bf16_t* vp = a.v + (int64_t)kstart * a.v_row + blk.kvh * a.v_head;
    PackedTiles<DH, NW> st;
    st.init(wave, lane, a.dim, a.k_row, a.v_row);
    const int64_t k_step = 64 * a.k_row, v_step = 64 * a.v_row;
    auto load = [&](int t) {                                                    // (called for t = 0, 1, 2 ..)
        char* to = smem + (t & 1) * 2 * G::TILE;
        st.load(wave, kp, seq_bytes_left(klen - t * 64, a.k_row * 2, a.dim), to, vp, seq_bytes_left(klen - t * 64, a.v_row * 2, a.dim), to + G::TILE);
        kp += k_step;
        vp += v_step;
    };
    PackedLane<DH> at;
    at.init(lane);

    if (ntile > 0) load(0);
    for (int t = 0; t < ntile; ++t) {
        char* kt_ = smem + (t & 1) * 2 * G::TILE;
        char* vt_ = kt_ + G::TILE;
        st.land(kt_, vt_);
        __syncthreads();
        if (t + 1 < ntile) load(t + 1);
        const int k0 = t * 64;
        if (k0 >= w_end) continue;
        at.forget();
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            f32x16_t sacc = packed_splat(0.f), dp = packed_splat(-delta);
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.row_frag(kt_ + kt * 32 * G::PITCH, ks), qf[ks], sacc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.row_frag(vt_ + kt * 32 * G::PITCH, ks), gf[ks], dp, 0, 0, 0);
            }
            if (k0 + 64 > klen || k0 + 63 > q0 + shift) {
                int lim = min(klen, qi + shift + 1) - k0 - 32 * kt - 4 * h;
                asm volatile("" : "+v"(lim));
#pragma unroll
                for (int r = 0; r < 16; ++r) sacc[r] = seq_crow(r) < lim ? sacc[r] : -INFINITY;
            }
            bf16x8_t ds[2];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = 8 * s2 + e;
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[r], c2, -lse2)) * dp[r];
                }
                ds[s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < G::DT; ++d)
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.tr_frag(kt_ + (kt * 2 + s2) * 16 * G::PITCH, d), ds[s2], acc[d], 0, 0, 0);
        }
    }
    __syncthreads();
    if (q0 < s.len)
        packed_write_rows<DH>(smem + wave * 32 * G::PITCH, acc, a.scale, a.dq + ((int64_t)(s.start + q0) * a.hq + blk.head) * a.dim, (int64_t)a.hq * a.dim,
                              min(32, s.len - q0), a.dim);
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

template <int DH>
static int packed_fwd_dispatch(PackedArgs& a, void* stream) {
    constexpr int NW = 4;
    a.nslots = a.rows_q / (32 * NW) + a.nseq + 1;
    return packed_launch(packed_fwd_kernel<DH, NW>, a, (int64_t)a.nslots * a.hq, 64 * NW, 4 * PackedGeo<DH>::TILE, stream);
}

template <int DH>
static int packed_bwd_dispatch(PackedArgs& a, void* stream) {
    constexpr int NW = 4;
    a.nslots = a.rows_q / (32 * NW) + a.nseq + 1;
    const int rc = packed_launch(packed_dq_kernel<DH, NW>, a, (int64_t)a.nslots * a.hq, 64 * NW, 4 * PackedGeo<DH>::TILE, stream);
    if (rc != GENIE_OK) return rc;
    return packed_dkv_run(a, stream);
}

extern "C" int genie_packed_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int32_t* cu_q, const int32_t* cu_k, int nseq,
                                          int rows_q, int rows_k, int hq, int hkv, int dim, const int64_t* q_strides, const int64_t* k_strides,
                                          const int64_t* v_strides, float scale, void* stream) {
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides, "genie_packed_attention_fwd: null strides");
    PackedArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.out = (bf16_t*)out; a.lse = lse;
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

extern "C" int genie_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, float* ws, int64_t ws_floats, void* dq,
                                          void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, int nseq, int rows_q, int rows_k, int hq, int hkv, int dim,
                                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* dout_strides, float scale,
                                          void* stream) {
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides && dout_strides, "genie_packed_attention_bwd: null strides");
    PackedArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.o = (const bf16_t*)out; a.dout = (const bf16_t*)dout;
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.lse = const_cast<float*>(lse); a.delta = ws;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseq = nseq; a.rows_q = rows_q; a.rows_k = rows_k; a.hq = hq; a.hkv = hkv; a.dim = dim; a.scale = scale;
    a.q_row = q_strides[0]; a.q_head = q_strides[1]; a.k_row = k_strides[0]; a.k_head = k_strides[1]; a.v_row = v_strides[0]; a.v_head = v_strides[1];
    a.g_row = dout_strides[0]; a.g_head = dout_strides[1];
    const int rc = packed_check("genie_packed_attention_bwd", a);
    if (rc != GENIE_OK) return rc;
    GENIE_CHECK_ARG(out && dout && lse && ws && dq && dk && dv, "genie_packed_attention_bwd: null pointer");
    GENIE_CHECK_ARG(ws_floats >= genie_packed_attention_bwd_ws_floats(nseq, rows_q, rows_k, hq, hkv, dim) && (uintptr_t)ws % 16 == 0,
                    "genie_packed_attention_bwd: workspace too small or not 16-byte aligned");
    if (dim <= 32) return packed_bwd_dispatch<32>(a, stream);
    if (dim <= 64) return packed_bwd_dispatch<64>(a, stream);
    if (dim <= 96) return packed_bwd_dispatch<96>(a, stream);
    return packed_bwd_dispatch<128>(a, stream);
}
