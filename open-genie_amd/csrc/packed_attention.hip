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
#include "seq_common.h"
#include "genie_hip.h"

struct PackedArgs {
    const bf16_t *q, *k, *v, *o, *dout;
    bf16_t *out, *dq, *dk, *dv;
    float* lse;                    // [Hq][rows_q]  log-sum-exp of the scaled scores, -inf where a row sees nothing
    float* delta;                  // [Hq][rows_q]  rowsum(dO o O), written by the dQ kernel for the dK / dV kernel
    const int32_t *cu_q, *cu_k;
    int nseq, rows_q, rows_k, hq, hkv, dim, nslots;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head;      // element strides (g: dO)
    float scale;
};

template <int DH>
struct PackedGeo {
    static constexpr int CPR = DH / 8;                              // 16-B chunks per row that are staged
    static constexpr int PITCH = DH <= 64 ? 128 : 256;              // LDS row pitch in bytes
    static constexpr int SW = PITCH / 16;                           // chunks of a pitch: the swizzle's range
    static constexpr int KS = DH / 16, DT = DH / 32;
    static constexpr int TILE = 64 * PITCH;
};

// byte offset of 16-B chunk `chunk` of row `row` inside a staged tile
template <int DH>
__device__ __forceinline__ uint32_t packed_at(int row, int chunk) {
    return (uint32_t)(row * PackedGeo<DH>::PITCH + (attn_swz<PackedGeo<DH>::SW>(row, chunk) << 4));
}

// Lane offsets of the two transposing reads that make one 32 x 16 operand fragment of the transposed tile: rows 4 h + 0..3 and 8 + 4 h + 0..3 of a
// 16-row step, columns 32 d + (lane & 31).  The swizzle's keys use row bits 0..3 only, so a step of 16 rows is a constant byte offset.
template <int DH>
__device__ __forceinline__ void packed_tr_offsets(uint32_t (&off)[PackedGeo<DH>::DT][2], int lane) {
    const int g16 = lane >> 4, rr = (lane >> 2) & 3, qq = lane & 3;
    const int r0 = 4 * (g16 >> 1) + rr;
#pragma unroll
    for (int d = 0; d < PackedGeo<DH>::DT; ++d) {
        const int col = d * 32 + 16 * (g16 & 1) + 4 * qq;
        off[d][0] = packed_at<DH>(r0, col >> 3) + (col & 7) * 2;
        off[d][1] = packed_at<DH>(r0 + 8, col >> 3) + (col & 7) * 2;
    }
}
__device__ __forceinline__ bf16x8_t packed_tr_frag(const char* tile, uint32_t o0, uint32_t o1) {
    const bf16x4_t lo = seq_tr16(tile + o0), hi = seq_tr16(tile + o1);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A pair of 64-row tiles (K and V, or Q and dO) on its way from memory to LDS.
template <int DH, int NT>
struct PackedStage {
    using G = PackedGeo<DH>;
    static constexpr int PIECES = 64 * G::CPR / NT;
    static_assert(64 * G::CPR % NT == 0, "every thread stages the same number of pieces");
    uint32_t va[PIECES], vb[PIECES], lds[PIECES];
    u32x4_t ra[PIECES], rb[PIECES];
    __device__ __forceinline__ void init(int tid, int dim, int64_t stride_a, int64_t stride_b) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int idx = tid + i * NT, row = idx / G::CPR, c = idx % G::CPR;
            const bool has = c * 8 < dim;
            va[i] = has ? (uint32_t)(row * stride_a * 2) + c * 16 : SEQ_OOB;
            vb[i] = has ? (uint32_t)(row * stride_b * 2) + c * 16 : SEQ_OOB;
            lds[i] = packed_at<DH>(row, c);
        }
    }
    __device__ __forceinline__ void load(const bf16_t* a, int left_a, const bf16_t* b, int left_b) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            ra[i] = seq_load16(a, left_a, va[i]);
            rb[i] = seq_load16(b, left_b, vb[i]);
        }
    }
    __device__ __forceinline__ void store(char* ta, char* tb) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            *reinterpret_cast<u32x4_t*>(ta + lds[i]) = ra[i];
            *reinterpret_cast<u32x4_t*>(tb + lds[i]) = rb[i];
        }
    }
};

// (slot, head) of a block.  Slots in descending order: the tiles with the most keys start first.  Heads fastest, key heads before the query heads that
// share them: consecutive blocks go round-robin over the 8 XCDs, so with 8, 4, 2 or 1 key heads an XCD's L2 sees one key head only.
struct PackedBlock { int slot, head, kvh; };
__device__ __forceinline__ PackedBlock packed_block(const PackedArgs& a, int nh) {
    PackedBlock b;
    const int id = (int)blockIdx.x, hi = id % nh;
    b.slot = a.nslots - 1 - id / nh;
    b.kvh = hi % a.hkv;
    b.head = b.kvh * (nh / a.hkv) + hi / a.hkv;
    return b;
}

// rows of `dst` (heads x dim, contiguous) behind the last sequence get zeros
template <int BM, int NT>
__device__ __forceinline__ void packed_zero_rows(bf16_t* dst, int heads, int dim, const SeqSlot& s, int head) {
    const int n = min(BM, s.len - s.tile * BM), cpr = dim / 8;
    for (int i = threadIdx.x; i < n * cpr; i += NT) {
        const long long row = s.start + s.tile * BM + i / cpr;
        *reinterpret_cast<u32x4_t*>(dst + (row * heads + head) * dim + (i % cpr) * 8) = u32x4_t{0, 0, 0, 0};
    }
}

// 32 rows of a wave's transposed accumulators (column = row of the output) to memory as 16-B chunks, by way of the wave's own 32 x PITCH LDS region:
// straight from the registers a store instruction would touch 32 rows with 8 B each.
template <int DH>
__device__ __forceinline__ void packed_write_rows(char* region, const f32x16_t (&acc)[PackedGeo<DH>::DT], float mul, bf16_t* dst, int64_t row_stride, int rows,
                                                  int dim) {
    using G = PackedGeo<DH>;
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const u32x2_t w = {pack_bf16x2(acc[d][4 * g] * mul, acc[d][4 * g + 1] * mul), pack_bf16x2(acc[d][4 * g + 2] * mul, acc[d][4 * g + 3] * mul)};
            *reinterpret_cast<u32x2_t*>(region + packed_at<DH>(c, 4 * d + g) + 8 * h) = w;
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < G::CPR / 2; ++i) {
        const int idx = i * 64 + lane, row = idx / G::CPR, ch = idx % G::CPR;
        if (row < rows && ch * 8 < dim)
            *reinterpret_cast<u32x4_t*>(dst + row * row_stride + ch * 8) = *reinterpret_cast<const u32x4_t*>(region + packed_at<DH>(row, ch));
    }
}

// this lane's row of a (rows x dim) matrix as MFMA operand fragments: 8 consecutive values of 16-wide step ks from column 16 ks + 8 h on
template <int DH>
__device__ __forceinline__ void packed_row_frags(bf16x8_t (&f)[PackedGeo<DH>::KS], const bf16_t* row, bool live, int dim) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ks = 0; ks < PackedGeo<DH>::KS; ++ks) {
        f[ks] = bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0};
        if (live && ks * 16 + h * 8 < dim) f[ks] = *reinterpret_cast<const bf16x8_t*>(row + ks * 16 + h * 8);
    }
}

__device__ __forceinline__ f32x16_t packed_splat(float v) {
    f32x16_t x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = v;
    return x;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Forward.  Online softmax in the exp2 domain with fp32 maximum, sum and accumulator; P is rounded to bf16 (at most 2^-8 of a weight, the precision
// of V itself) because the second product runs on the matrix cores.  The running maximum is "sum-triggered": a tile is exponentiated against the
// maximum as it stands, and only a lane whose partial row sum passes 2^8 (inf and NaN too) has the tile redone with its exact maximum -- no
// per-tile maximum tree in the steady state.  The first tile always takes its maximum, and every row that sees any key sees key 0.
// ------------------------------------------------------------------------------------------------------------------------------
template <int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? 3 : 2) packed_fwd_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    constexpr int BM = 32 * NW, NT = 64 * NW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const PackedBlock blk = packed_block(a, a.hq);
    const SeqSlot s = seq_find<BM>(a.cu_q, a.nseq, a.rows_q, blk.slot);
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
    PackedStage<DH, NT> st;
    st.init(tid, a.dim, a.k_row, a.v_row);
    auto load = [&](int t) {
        st.load(kp + (int64_t)t * 64 * a.k_row, seq_bytes_left(klen - t * 64, a.k_row * 2, a.dim), vp + (int64_t)t * 64 * a.v_row,
                seq_bytes_left(klen - t * 64, a.v_row * 2, a.dim));
    };
    uint32_t k_off[G::KS], v_off[G::DT][2];
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) k_off[ks] = packed_at<DH>(lane & 31, ks * 2 + h);
    packed_tr_offsets<DH>(v_off, lane);

    if (ntile > 0) load(0);
    for (int t = 0; t < ntile; ++t) {
        char* kt_ = smem + (t & 1) * 2 * G::TILE;
        char* vt_ = kt_ + G::TILE;
        st.store(kt_, vt_);
        __syncthreads();
        if (t + 1 < ntile) load(t + 1);
        const int k0 = t * 64;
        if (k0 >= w_end) continue;                                              // (wave-uniform) nothing of this tile is visible to these 32 rows
        bool with_max = t == 0;
        bf16x8_t pf[4];
        float psum;
        for (;;) {
            f32x16_t sacc[2] = {packed_splat(0.f), packed_splat(0.f)};
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    sacc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(kt_ + kt * 32 * G::PITCH + k_off[ks]), qf[ks], sacc[kt],
                                                                       0, 0, 0);
            if (k0 + 64 > klen || k0 + 63 > q0 + shift) {                       // the tile crosses the last key or the diagonal of these rows
                const int lim = min(klen, qi + shift + 1) - k0 - 4 * h;
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
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
                oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(packed_tr_frag(vt_ + ks * 16 * G::PITCH, v_off[d][0], v_off[d][1]), pf[ks], oacc[d], 0, 0, 0);
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
    const SeqSlot s = seq_find<BM>(a.cu_q, a.nseq, a.rows_q, blk.slot);
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
    PackedStage<DH, NT> st;
    st.init(tid, a.dim, a.k_row, a.v_row);
    auto load = [&](int t) {
        st.load(kp + (int64_t)t * 64 * a.k_row, seq_bytes_left(klen - t * 64, a.k_row * 2, a.dim), vp + (int64_t)t * 64 * a.v_row,
                seq_bytes_left(klen - t * 64, a.v_row * 2, a.dim));
    };
    uint32_t k_off[G::KS], t_off[G::DT][2];
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) k_off[ks] = packed_at<DH>(lane & 31, ks * 2 + h);
    packed_tr_offsets<DH>(t_off, lane);

    if (ntile > 0) load(0);
    for (int t = 0; t < ntile; ++t) {
        char* kt_ = smem + (t & 1) * 2 * G::TILE;
        char* vt_ = kt_ + G::TILE;
        st.store(kt_, vt_);
        __syncthreads();
        if (t + 1 < ntile) load(t + 1);
        const int k0 = t * 64;
        if (k0 >= w_end) continue;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            f32x16_t sacc = packed_splat(0.f), dp = packed_splat(-delta);
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(kt_ + kt * 32 * G::PITCH + k_off[ks]), qf[ks], sacc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(vt_ + kt * 32 * G::PITCH + k_off[ks]), gf[ks], dp, 0, 0, 0);
            }
            const bool edge = k0 + 64 > klen || k0 + 63 > q0 + shift;
            const int lim = min(klen, qi + shift + 1) - k0 - 4 * h;
            bf16x8_t ds[2];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = 8 * s2 + e;
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[r], c2, -lse2)) * dp[r];
                    if (edge) x[e] = kt * 32 + seq_crow(r) < lim ? x[e] : 0.f;
                }
                ds[s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < G::DT; ++d)
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(packed_tr_frag(kt_ + (kt * 2 + s2) * 16 * G::PITCH, t_off[d][0], t_off[d][1]), ds[s2], acc[d],
                                                                     0, 0, 0);
        }
    }
    __syncthreads();
    if (q0 < s.len)
        packed_write_rows<DH>(smem + wave * 32 * G::PITCH, acc, a.scale, a.dq + ((int64_t)(s.start + q0) * a.hq + blk.head) * a.dim, (int64_t)a.hq * a.dim,
                              min(32, s.len - q0), a.dim);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Backward, dK and dV: one wave owns 32 keys of one key head and walks the query rows that see them, head after head of the group -- the sum over the
// group's heads happens in the accumulators, in a fixed order.  S = Q K^T (lane = key): P and dS are again operand-shaped for dV^T = dO^T P and
// dK^T = Q^T dS.  The rows' log-sum-exp and delta run along the accumulator's rows and are read from LDS beside the tile.
// ------------------------------------------------------------------------------------------------------------------------------
template <int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? 2 : 1) packed_dkv_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    constexpr int BN = 32 * NW, NT = 64 * NW, STAGE = 2 * G::TILE + 512;
    static_assert(NT >= 128, "the first 128 threads fetch the rows' statistics");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int kvh = (int)blockIdx.x % a.hkv, slot = (int)blockIdx.x / a.hkv, group = a.hq / a.hkv;        // ascending: the first keys are seen by most rows
    const SeqSlot s = seq_find<BN>(a.cu_k, a.nseq, a.rows_k, slot);
    if (s.tile < 0 || s.tile * BN >= s.len) return;
    if (s.seq == a.nseq) {
        packed_zero_rows<BN, NT>(a.dk, a.hkv, a.dim, s, kvh);
        packed_zero_rows<BN, NT>(a.dv, a.hkv, a.dim, s, kvh);
        return;
    }
    const int qstart = seq_cu(a.cu_q, s.seq, a.rows_q), qlen = max(0, seq_cu(a.cu_q, s.seq + 1, a.rows_q) - qstart);
    const int shift = s.len - qlen;                                             // key j is seen by rows i >= j - shift
    const int j0 = s.tile * BN + wave * 32, kj = j0 + (lane & 31);
    const int first = max(0, s.tile * BN - shift) & ~63;                        // first query row the block needs, on a tile border
    const int w_first = j0 - shift;
    const int tiles = max(0, (qlen - first + 63) >> 6), steps = tiles * group;

    bf16x8_t kf[G::KS], vf[G::KS];
    const int64_t krow = s.start + kj;
    packed_row_frags<DH>(kf, a.k + krow * a.k_row + kvh * a.k_head, kj < s.len, a.dim);
    packed_row_frags<DH>(vf, a.v + krow * a.v_row + kvh * a.v_head, kj < s.len, a.dim);
    f32x16_t dk[G::DT], dv[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) dk[d] = dv[d] = packed_splat(0.f);
    const float c2 = a.scale * 1.4426950408889634f;

    PackedStage<DH, NT> st;
    st.init(tid, a.dim, a.q_row, a.g_row);
    float stat = 0.f;                                                           // threads 0..63: -lse * log2 e, 64..127: -delta of the tile's rows
    auto load = [&](int i) {
        const int head = kvh * group + i / tiles, r0 = first + (i % tiles) * 64;
        const bf16_t* qp = a.q + (int64_t)(qstart + r0) * a.q_row + head * a.q_head;
        const bf16_t* gp = a.dout + (int64_t)(qstart + r0) * a.g_row + head * a.g_head;
        st.load(qp, seq_bytes_left(qlen - r0, a.q_row * 2, a.dim), gp, seq_bytes_left(qlen - r0, a.g_row * 2, a.dim));
        if (tid < 128) {
            const int row = r0 + (tid & 63);
            const int64_t at = (int64_t)head * a.rows_q + qstart + row;
            stat = tid < 64 ? -INFINITY : 0.f;
            if (row < qlen) {
                const float x = tid < 64 ? a.lse[at] : a.delta[at];
                stat = tid >= 64 ? -x : (x == -INFINITY ? -INFINITY : -x * 1.4426950408889634f);
            }
        }
    };
    uint32_t r_off[G::KS], t_off[G::DT][2];
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) r_off[ks] = packed_at<DH>(lane & 31, ks * 2 + h);
    packed_tr_offsets<DH>(t_off, lane);

    if (steps > 0) load(0);
    for (int i = 0; i < steps; ++i) {
        char* qt_ = smem + (i & 1) * STAGE;
        char* gt_ = qt_ + G::TILE;
        float* stats = reinterpret_cast<float*>(gt_ + G::TILE);
        st.store(qt_, gt_);
        if (tid < 128) stats[tid] = stat;
        __syncthreads();
        if (i + 1 < steps) load(i + 1);
        const int r0 = first + (i % tiles) * 64;
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
            const int rbase = r0 + qt * 32;
            if (rbase + 31 < w_first || rbase >= qlen) continue;                // (wave-uniform) no row of these 32 sees this wave's keys
            f32x16_t sacc = packed_splat(0.f), dp, l2;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(stats + qt * 32 + 8 * g + 4 * h), y = *reinterpret_cast<const f32x4_t*>(stats + 64 + qt * 32 + 8 * g + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) { l2[4 * g + e] = x[e]; dp[4 * g + e] = y[e]; }
            }
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(qt_ + qt * 32 * G::PITCH + r_off[ks]), kf[ks], sacc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(gt_ + qt * 32 * G::PITCH + r_off[ks]), vf[ks], dp, 0, 0, 0);
            }
            const bool edge = rbase < j0 + 31 - shift;                          // some row of these 32 does not see all of the 32 keys
            const int lim = kj - shift - rbase - 4 * h;                         // rows below do not see this lane's key
            bf16x8_t pf[2], ds[2];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                float p[8], x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = 8 * s2 + e;
                    p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[r], c2, l2[r]));
                    x[e] = p[e] * dp[r];
                    if (edge) {
                        const bool sees = seq_crow(r) >= lim;
                        p[e] = sees ? p[e] : 0.f;
                        x[e] = sees ? x[e] : 0.f;
                    }
                }
                pf[s2] = seq_pack8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
                ds[s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < G::DT; ++d) {
                    dv[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(packed_tr_frag(gt_ + (qt * 2 + s2) * 16 * G::PITCH, t_off[d][0], t_off[d][1]), pf[s2], dv[d], 0, 0, 0);
                    dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(packed_tr_frag(qt_ + (qt * 2 + s2) * 16 * G::PITCH, t_off[d][0], t_off[d][1]), ds[s2], dk[d], 0, 0, 0);
                }
        }
    }
    __syncthreads();
    if (j0 < s.len) {
        const int64_t at = ((int64_t)(s.start + j0) * a.hkv + kvh) * a.dim;
        char* region = smem + wave * 64 * G::PITCH;
        packed_write_rows<DH>(region, dk, a.scale, a.dk + at, (int64_t)a.hkv * a.dim, min(32, s.len - j0), a.dim);
        packed_write_rows<DH>(region + 32 * G::PITCH, dv, 1.f, a.dv + at, (int64_t)a.hkv * a.dim, min(32, s.len - j0), a.dim);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// C entry points
// ------------------------------------------------------------------------------------------------------------------------------
static int packed_check(const char* what, const PackedArgs& a) {
    GENIE_CHECK_ARG(a.q && a.k && a.v && a.cu_q && a.cu_k, "%s: null pointer", what);
    GENIE_CHECK_ARG(a.nseq >= 0 && a.rows_q >= 0 && a.rows_k >= 0, "%s: negative size", what);
    GENIE_CHECK_ARG(a.hkv > 0 && a.hq > 0 && a.hq % a.hkv == 0, "%s: %d query heads are no multiple of %d key heads", what, a.hq, a.hkv);
    GENIE_CHECK_ARG(a.dim > 0 && a.dim % 8 == 0 && a.dim <= 128, "%s: head width %d (a multiple of 8 up to 128 is supported)", what, a.dim);
    GENIE_CHECK_ARG(a.scale > 0.f && a.scale < 1e30f, "%s: scale must be positive and finite", what);
    const int64_t s[8] = {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.g_row, a.g_head};
    for (int i = 0; i < 8; ++i) GENIE_CHECK_ARG(s[i] >= 0 && s[i] % 8 == 0, "%s: strides must be multiples of 8 elements", what);
    for (int i = 0; i < 8; i += 2)
        GENIE_CHECK_ARG(s[i] >= a.dim && s[i] < (1 << 21), "%s: row stride %lld (the head width up to 2^21 elements is supported)", what, (long long)s[i]);
    return GENIE_OK;
}

template <typename K>
static int packed_launch(K kernel, const PackedArgs& a, int64_t blocks, int threads, int lds, void* stream) {
    GENIE_CHECK_ARG(blocks < (1ll << 31), "packed attention: too many blocks");
    if (blocks <= 0) return GENIE_OK;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) {
            genie_set_error("packed attention: %s", hipGetErrorString(e));
            return GENIE_ERR_HIP;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, (hipStream_t)stream, a);
    GENIE_CHECK_LAUNCH();
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
    a.nslots = a.rows_k / (32 * NW) + a.nseq + 1;
    return packed_launch(packed_dkv_kernel<DH, NW>, a, (int64_t)a.nslots * a.hkv, 64 * NW, 4 * PackedGeo<DH>::TILE + 1024, stream);
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

extern "C" int genie_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, float* delta_ws, void* dq,
                                          void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, int nseq, int rows_q, int rows_k, int hq, int hkv, int dim,
                                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* dout_strides, float scale,
                                          void* stream) {
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides && dout_strides, "genie_packed_attention_bwd: null strides");
    PackedArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.o = (const bf16_t*)out; a.dout = (const bf16_t*)dout;
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.lse = const_cast<float*>(lse); a.delta = delta_ws;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseq = nseq; a.rows_q = rows_q; a.rows_k = rows_k; a.hq = hq; a.hkv = hkv; a.dim = dim; a.scale = scale;
    a.q_row = q_strides[0]; a.q_head = q_strides[1]; a.k_row = k_strides[0]; a.k_head = k_strides[1]; a.v_row = v_strides[0]; a.v_head = v_strides[1];
    a.g_row = dout_strides[0]; a.g_head = dout_strides[1];
    const int rc = packed_check("genie_packed_attention_bwd", a);
    if (rc != GENIE_OK) return rc;
    GENIE_CHECK_ARG(out && dout && lse && delta_ws && dq && dk && dv, "genie_packed_attention_bwd: null pointer");
    if (dim <= 32) return packed_bwd_dispatch<32>(a, stream);
    if (dim <= 64) return packed_bwd_dispatch<64>(a, stream);
    if (dim <= 96) return packed_bwd_dispatch<96>(a, stream);
    return packed_bwd_dispatch<128>(a, stream);
}
