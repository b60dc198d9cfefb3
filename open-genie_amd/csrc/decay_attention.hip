// Linear attention with a decay for each head over packed sequences (chunked form, forward and backward) and its recurrence for single tokens.
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   l = exp(log_decay[head])                (S: d_k x d_v, fp32)
//
// The forward and the three gradients are ONE form,  y_t = scale sum_{s <= t} l^(t-s) (a_t . b_s) c_s :
//   o = form(q, k, v)   dq = form(do, v, k)   and, run from the sequence's end,   dv = form(k, q, do)   dk = form(v, do, q)
// with the state M = sum l^.. b_s c_s^T (for dq the transpose of the forward's, for dk that of dv's).  Chunks of 64 tokens:
//   y = l^(t+1) a_t M + (A B^T o D) C,  D_ts = l^(t-s) for s <= t;     M <- l^64 M + sum_s l^(63-s) b_s c_s^T
// All powers have exponents >= 0 (strong decays underflow to 0, nothing overflows).
//
// A block walks one SEGMENT of a sequence for one head; wave w owns columns 32 w .. 32 w + 31 of C, of the output and of M, which lives in its
// accumulators: as the bf16 operand of a M it needs no exchange, because the accumulator layout is the operand layout up to an order of the
// contraction index, and A and B are staged in that order.  Long sequences are cut into segments so that few sequences still fill 256 CUs: the segments'
// own states first (B and C only), an elementwise scan over them, then all segments at once.
//
// Roundings to bf16: the scores and M as matrix operands of an output that is itself rounded to bf16 (M itself stays fp32).  The state update must not
// round its decayed operand, because the state is an fp32 result that lives on: l^(63-s) c_s goes in as a sum of two bf16 values (2^-16 left).
#include "seq_common.h"
#include "genie_hip.h"

struct DecayRole {
    const bf16_t *a, *b, *c;
    bf16_t* y;                                   // [rows][heads][dc]
    int64_t a_row, a_head, b_row, b_head, c_row, c_head;
    int da, dc, reverse;
    int m_a, m_c;                                // element strides of M inside a stored matrix (the transposed use swaps them)
    const float* seq_state;                      // state in front of each sequence, [nseq][heads][matrix], or NULL
    float* seg_state;                            // [slot][heads][matrix]: state in front of every segment but a sequence's first
    float* final_state;                          // [nseq][heads][da][dc], or NULL
};
struct DecayArgs {
    DecayRole r[3];
    const int32_t* cu;
    const float* log_decay;
    int nseq, rows, heads, seg, nslots;
    float scale;
};

template <int DH>
struct DecayGeo {
    static constexpr int NW = DH / 32, NT = 64 * NW, CPR = DH / 8, PITCH = DH <= 64 ? 128 : 256, SW = PITCH / 16, KS = DH / 16, DT = DH / 32;
    static constexpr int TILE = 64 * PITCH, PIECES = 4;
};

// l^e for e >= 0 (l = 0 included: l^0 = 1)
__device__ __forceinline__ float decay_pow(float log2_l, int e) { return e == 0 ? 1.f : __builtin_amdgcn_exp2f(log2_l * (float)e); }

// One 64-token tile of a matrix from memory into registers and on to LDS.  A chunk with nv < 64 tokens (a sequence's last) sits in the tile's LAST rows, so that
// the weights towards the chunk's end, l^(63-s), hold for it too; the rows in front of it read zeros: their offsets wrap past any range (forward) or lie
// behind the last token (reverse, where row i of the tile is the token 63 - i rows up in memory).
// ORDERED: inside each 16 columns the four 8-B pieces are stored in the order 0, 2, 1, 3, so that a lane half's 16 B are columns 4 h .. 4 h + 3 and
// 8 + 4 h .. 8 + 4 h + 3 -- the accumulator layout's rows.
// A thread's four pieces are 16 rows apart in one column chunk (the swizzle's keys use row bits 0..3: one LDS address and constant offsets).
template <int DH, bool ORDERED>
struct DecayTile {
    using G = DecayGeo<DH>;
    static_assert(G::NT / G::CPR == 16 && G::NT % G::CPR == 0, "pieces are 16 rows apart");
    uint32_t off, lds0, lds1;
    int step;
    u32x4_t r[G::PIECES];
    const bf16_t* base;
    int64_t row;
    int dim;
    bool rev;
    __device__ __forceinline__ void init(int tid, const bf16_t* first, int64_t stride, int width, bool reverse) {
        base = first; row = stride; dim = width; rev = reverse;
        const int rr = tid / G::CPR, c = tid % G::CPR;
        off = c * 8 < dim ? (uint32_t)((reverse ? 63 - rr : rr) * stride * 2) + c * 16 : SEQ_OOB;
        step = (int)(reverse ? -32 * stride : 32 * stride);
        if (c * 8 >= dim) step = 0;
        if (ORDERED) {
            lds0 = (uint32_t)(rr * G::PITCH + (attn_swz<G::SW>(rr, c & ~1) << 4) + (c & 1) * 8);
            lds1 = (uint32_t)(rr * G::PITCH + (attn_swz<G::SW>(rr, c | 1) << 4) + (c & 1) * 8);
        } else {
            lds0 = (uint32_t)(rr * G::PITCH + (attn_swz<G::SW>(rr, c) << 4));
        }
    }
    // the chunk of tokens p .. p + nv - 1 of the walk over a sequence of len tokens (reverse: counted from its end)
    __device__ __forceinline__ void load(int p, int len) {
        const int nv = min(64, len - p);
        const bf16_t* t = base + (int64_t)(rev ? len - p - nv : p) * row;
        const int left = seq_bytes_left(nv, row * 2, dim);
        const uint32_t o = off - (rev ? 0u : (uint32_t)((64 - nv) * row * 2));
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) r[i] = seq_load16(t, left, o + (uint32_t)(i * step));
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) {
            if constexpr (ORDERED) {
                *reinterpret_cast<u32x2_t*>(tile + lds0 + i * 16 * G::PITCH) = u32x2_t{r[i][0], r[i][1]};
                *reinterpret_cast<u32x2_t*>(tile + lds1 + i * 16 * G::PITCH) = u32x2_t{r[i][2], r[i][3]};
            } else {
                *reinterpret_cast<u32x4_t*>(tile + lds0 + i * 16 * G::PITCH) = r[i];
            }
        }
    }
};

// lane offset of a transposing read of columns col0 + (lane & 31), rows 4 h + 0..3 (+ 8 rows: second = true) of a 16-row step
template <int DH, bool ORDERED>
__device__ __forceinline__ uint32_t decay_tr_offset(int lane, int col0, bool second) {
    using G = DecayGeo<DH>;
    const int g16 = lane >> 4, row = 4 * (g16 >> 1) + ((lane >> 2) & 3) + (second ? 8 : 0);
    const int piece = (col0 + 16 * (g16 & 1) + 4 * (lane & 3)) >> 2;
    int chunk = piece >> 1, half = piece & 1;
    if (ORDERED) { const int c = chunk; chunk = (c & ~1) + half; half = c & 1; }
    return (uint32_t)(row * G::PITCH + (attn_swz<G::SW>(row, chunk) << 4) + half * 8);
}
__device__ __forceinline__ bf16x8_t decay_tr(const char* tile, uint32_t o0, uint32_t o1) {
    const bf16x4_t lo = seq_tr16(tile + o0), hi = seq_tr16(tile + o1);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// M <- all M + sum_s l^(63-s) b_s c_s^T over a staged chunk (cf: this wave's 32 columns of C, transposed fragments).
// fade[r] = l^(31 - row r of a 32-row half), p32 = l^32.
template <int DH>
__device__ __forceinline__ void decay_update(f32x16_t (&m)[DecayGeo<DH>::DT], const char* bt, const uint32_t (&boff)[DecayGeo<DH>::DT][2], const bf16x8_t (&cf)[4],
                                             float all, const float (&fade)[16], float p32) {
    using G = DecayGeo<DH>;
#pragma unroll
    for (int i = 0; i < G::DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[i][r] *= all;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        float hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi[j] = bf16_to_f32((bf16_t)cf[ks][j]) * fade[8 * (ks & 1) + j];
            if (ks < 2) hi[j] *= p32;
        }
        const u32x4_t fh = {pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]), pack_bf16x2(hi[4], hi[5]), pack_bf16x2(hi[6], hi[7])};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[2 * j] = hi[2 * j] - __uint_as_float(fh[j] << 16);
            lo[2 * j + 1] = hi[2 * j + 1] - __uint_as_float(fh[j] & 0xffff0000u);
        }
        const bf16x8_t fl = seq_pack8(lo[0], lo[1], lo[2], lo[3], lo[4], lo[5], lo[6], lo[7]);
#pragma unroll
        for (int i = 0; i < G::DT; ++i) {
            const bf16x8_t bf = decay_tr(bt + ks * 16 * G::PITCH, boff[i][0], boff[i][1]);
            m[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf, __builtin_bit_cast(bf16x8_t, fh), m[i], 0, 0, 0);
            m[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf, fl, m[i], 0, 0, 0);
        }
    }
}

__device__ __forceinline__ f32x16_t decay_zero() {
    f32x16_t x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = 0.f;
    return x;
}

// The state each segment leaves behind when it starts from nothing (every segment but a sequence's last), into the slot AFTER its own.
template <int DH>
__global__ void __launch_bounds__(64 * (DH / 32), 2) decay_state_kernel(const DecayArgs g) {
    using G = DecayGeo<DH>;
    __shared__ __attribute__((aligned(16))) char smem[2 * G::TILE];
    const DecayRole& R = g.r[0];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int head = (int)blockIdx.x % g.heads, slot = (int)blockIdx.x / g.heads;
    const SeqSlot s = seq_find_n(g.cu, g.nseq, g.rows, g.seg, slot);
    if (s.seq == g.nseq || s.tile < 0 || (int64_t)(s.tile + 1) * g.seg >= s.len) return;
    const float log2_l = g.log_decay[head] * 1.4426950408889634f;
    float fade[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) fade[r] = decay_pow(log2_l, 31 - (seq_crow(r) + 4 * h));
    const float p32 = decay_pow(log2_l, 32);
    uint32_t boff[G::DT][2], coff[2];
#pragma unroll
    for (int i = 0; i < G::DT; ++i) { boff[i][0] = decay_tr_offset<DH, true>(lane, 32 * i, false); boff[i][1] = decay_tr_offset<DH, true>(lane, 32 * i, true); }
    coff[0] = decay_tr_offset<DH, false>(lane, 32 * wave, false);
    coff[1] = decay_tr_offset<DH, false>(lane, 32 * wave, true);
    DecayTile<DH, true> tb;
    DecayTile<DH, false> tc;
    tb.init(tid, R.b + (int64_t)s.start * R.b_row + head * R.b_head, R.b_row, R.da, R.reverse);
    tc.init(tid, R.c + (int64_t)s.start * R.c_row + head * R.c_head, R.c_row, R.dc, R.reverse);
    f32x16_t m[G::DT];
#pragma unroll
    for (int i = 0; i < G::DT; ++i) m[i] = decay_zero();
    const int p0 = s.tile * g.seg, p1 = p0 + g.seg;
    char *bt = smem, *ct = smem + G::TILE;
    tb.load(p0, s.len);
    tc.load(p0, s.len);
    for (int p = p0; p < p1; p += 64) {
        tb.store(bt);
        tc.store(ct);
        __syncthreads();
        if (p + 64 < p1) { tb.load(p + 64, s.len); tc.load(p + 64, s.len); }
        bf16x8_t cf[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) cf[ks] = decay_tr(ct + ks * 16 * G::PITCH, coff[0], coff[1]);
        decay_update<DH>(m, bt, boff, cf, p32 * p32, fade, p32);
        __syncthreads();
    }
    float* dst = R.seg_state + ((int64_t)(slot + 1) * g.heads + head) * R.da * R.dc;
    const int col = 32 * wave + (lane & 31);
    if (col < R.dc) {
#pragma unroll
        for (int i = 0; i < G::DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * i + seq_crow(r) + 4 * h;
                if (row < R.da) dst[(uint32_t)(row * R.dc + col)] = m[i][r];
            }
    }
}

// seg_state[first slot + i] <- l^seg (state in front of segment i - 1) + (what segment i - 1 adds), i = 1 ..: elementwise over the matrix, one thread per four
// elements, the next segments' values requested ahead of the chain.
__global__ void __launch_bounds__(256) decay_scan_kernel(const DecayArgs g, int matrix) {
    const DecayRole& R = g.r[0];
    const int seq = (int)blockIdx.x / g.heads, head = (int)blockIdx.x % g.heads;
    const int e = ((int)blockIdx.y * 256 + (int)threadIdx.x) * 4;
    if (e >= matrix) return;
    const int start = seq_cu(g.cu, seq, g.rows), len = max(0, seq_cu(g.cu, seq + 1, g.rows) - start);
    const int nseg = (len + g.seg - 1) / g.seg;
    if (nseg < 2) return;
    const float l = decay_pow(g.log_decay[head] * 1.4426950408889634f, g.seg);
    f32x4_t m = {0.f, 0.f, 0.f, 0.f};
    if (R.seq_state) m = *reinterpret_cast<const f32x4_t*>(R.seq_state + ((int64_t)seq * g.heads + head) * matrix + e);
    const int64_t step = (int64_t)g.heads * matrix;
    // first slot of the sequence; wrong cu contents can reach past the last slot: clamp
    const int s0 = start / g.seg + seq, last = min(nseg - 1, g.nslots - 1 - s0);
    float* p = R.seg_state + ((int64_t)(s0 + 1) * g.heads + head) * matrix + e;
    int i = 0;
    for (; i + 8 <= last; i += 8) {
        f32x4_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const f32x4_t*>(p + (i + j) * step);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int q = 0; q < 4; ++q) m[q] = __builtin_fmaf(m[q], l, x[j][q]);
            *reinterpret_cast<f32x4_t*>(p + (i + j) * step) = m;
        }
    }
    for (; i < last; ++i) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(p + i * step);
#pragma unroll
        for (int q = 0; q < 4; ++q) m[q] = __builtin_fmaf(m[q], l, x[q]);
        *reinterpret_cast<f32x4_t*>(p + i * step) = m;
    }
}

template <int DH>
__global__ void __launch_bounds__(64 * (DH / 32), 2) decay_sweep_kernel(const DecayArgs g) {
    using G = DecayGeo<DH>;
    __shared__ __attribute__((aligned(16))) char smem[4 * G::TILE];
    const DecayRole& R = g.r[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int head = (int)blockIdx.x % g.heads, slot = (int)blockIdx.x / g.heads;
    const int64_t matrix = (int64_t)R.da * R.dc;
    if (slot >= g.nslots) {                                                     // (launched when final states are asked for) sequences without tokens
        const int seq = slot - g.nslots;
        if (R.final_state && seq_cu(g.cu, seq + 1, g.rows) <= seq_cu(g.cu, seq, g.rows)) {
            const int64_t at = ((int64_t)seq * g.heads + head) * matrix;
            for (int i = tid; i < matrix; i += G::NT) R.final_state[at + i] = R.seq_state ? R.seq_state[at + i] : 0.f;
        }
        return;
    }
    const SeqSlot s = seq_find_n(g.cu, g.nseq, g.rows, g.seg, slot);
    const int p0 = s.tile * g.seg;
    if (s.tile < 0 || p0 >= s.len) return;
    const int p1 = min(s.len, p0 + g.seg), cpr = R.dc / 8;
    if (s.seq == g.nseq) {                                                      // rows behind the last sequence
        for (int i = tid; i < (p1 - p0) * cpr; i += G::NT)
            *reinterpret_cast<u32x4_t*>(R.y + ((int64_t)(s.start + p0 + i / cpr) * g.heads + head) * R.dc + (i % cpr) * 8) = u32x4_t{0, 0, 0, 0};
        return;
    }
    const float log2_l = g.log_decay[head] * 1.4426950408889634f;
    float near[16], fade[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int k = seq_crow(r) + 4 * h, d = (lane & 31) - k;                 // query - key inside a 32 x 32 tile on the diagonal
        near[r] = d >= 0 ? decay_pow(log2_l, max(0, d)) : 0.f;
        fade[r] = decay_pow(log2_l, 31 - k);
    }
    const float next = decay_pow(log2_l, (lane & 31) + 1), p32 = decay_pow(log2_l, 32);
    uint32_t roff[G::KS], boff[G::DT][2], coff[2];
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) roff[ks] = (uint32_t)((lane & 31) * G::PITCH + (attn_swz<G::SW>(lane & 31, 2 * ks + h) << 4));
#pragma unroll
    for (int i = 0; i < G::DT; ++i) { boff[i][0] = decay_tr_offset<DH, true>(lane, 32 * i, false); boff[i][1] = decay_tr_offset<DH, true>(lane, 32 * i, true); }
    coff[0] = decay_tr_offset<DH, false>(lane, 32 * wave, false);
    coff[1] = decay_tr_offset<DH, false>(lane, 32 * wave, true);

    f32x16_t m[G::DT];
    const float* init = p0 > 0 ? R.seg_state + ((int64_t)slot * g.heads + head) * matrix
                               : (R.seq_state ? R.seq_state + ((int64_t)s.seq * g.heads + head) * matrix : nullptr);
    const int mcol = 32 * wave + (lane & 31);
    // (clamped addresses and selects: a branch per element would make the compiler copy whole accumulators)
    const float keep = init && mcol < R.dc ? 1.f : 0.f;
    const float* from = init ? init : g.log_decay;
    const int mc_ = mcol < R.dc ? mcol * R.m_c : 0;
#pragma unroll
    for (int i = 0; i < G::DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = 32 * i + seq_crow(r) + 4 * h;
            const float x = from[(uint32_t)(init && row < R.da ? row * R.m_a + mc_ : 0)];
            m[i][r] = keep != 0.f && row < R.da ? x : 0.f;
        }

    DecayTile<DH, true> ta, tb;
    DecayTile<DH, false> tc;
    ta.init(tid, R.a + (int64_t)s.start * R.a_row + head * R.a_head, R.a_row, R.da, R.reverse);
    tb.init(tid, R.b + (int64_t)s.start * R.b_row + head * R.b_head, R.b_row, R.da, R.reverse);
    tc.init(tid, R.c + (int64_t)s.start * R.c_row + head * R.c_head, R.c_row, R.dc, R.reverse);
    const int orow = tid / G::CPR, ocol = (tid % G::CPR) * 8, oat = orow * G::PITCH + (attn_swz<G::SW>(orow, tid % G::CPR) << 4);
    char *at = smem, *bt = at + G::TILE, *ct = bt + G::TILE, *yt = ct + G::TILE;
    ta.load(p0, s.len);
    tb.load(p0, s.len);
    tc.load(p0, s.len);
    for (int p = p0; p < p1; p += 64) {
        ta.store(at);
        tb.store(bt);
        tc.store(ct);
        __syncthreads();
        const int nv = min(64, p1 - p), blank = 64 - nv;                        // tile rows in front of the chunk's first token
        const bool more = p + 64 < p1;
        if (more) {
            ta.load(p + 64, s.len);
            tb.load(p + 64, s.len);
            tc.load(p + 64, s.len);
        }
        bf16x8_t cf[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) cf[ks] = decay_tr(ct + ks * 16 * G::PITCH, coff[0], coff[1]);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            bf16x8_t af[G::KS];
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) af[ks] = *reinterpret_cast<const bf16x8_t*>(at + tt * 32 * G::PITCH + roff[ks]);
            f32x16_t y = decay_zero();
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                const int i = ks >> 1, r = 8 * (ks & 1);
                const bf16x8_t mf = seq_pack8(m[i][r], m[i][r + 1], m[i][r + 2], m[i][r + 3], m[i][r + 4], m[i][r + 5], m[i][r + 6], m[i][r + 7]);
                y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mf, af[ks], y, 0, 0, 0);
            }
            const float lead = decay_pow(log2_l, max(0, tt * 32 + (lane & 31) + 1 - blank));
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] *= lead;
#pragma unroll
            for (int st = 0; st <= tt; ++st) {
                f32x16_t x = decay_zero();
#pragma unroll
                for (int ks = 0; ks < G::KS; ++ks)
                    x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(bt + st * 32 * G::PITCH + roff[ks]), af[ks], x, 0, 0, 0);
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = x[8 * s2 + e] * (st == tt ? near[8 * s2 + e] : fade[8 * s2 + e] * next);
                    y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cf[2 * st + s2], seq_pack8(w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]), y, 0, 0, 0);
                }
            }
            // y^T (column = token) to the output tile, rows = tokens
            const int row = tt * 32 + (lane & 31);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x2_t w = {pack_bf16x2(y[4 * q] * g.scale, y[4 * q + 1] * g.scale), pack_bf16x2(y[4 * q + 2] * g.scale, y[4 * q + 3] * g.scale)};
                *reinterpret_cast<u32x2_t*>(yt + row * G::PITCH + (attn_swz<G::SW>(row, 4 * wave + q) << 4) + 8 * h) = w;
            }
        }
        decay_update<DH>(m, bt, boff, cf, nv == 64 ? p32 * p32 : decay_pow(log2_l, nv), fade, p32);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) {
            const int rr = orow + 16 * i, t = p + rr - blank;
            if (rr >= blank && ocol < R.dc) {
                const int64_t tok = s.start + (R.reverse ? s.len - 1 - t : t);
                *reinterpret_cast<u32x4_t*>(R.y + (tok * g.heads + head) * R.dc + ocol) = *reinterpret_cast<const u32x4_t*>(yt + oat + i * 16 * G::PITCH);
            }
        }
    }
    if (R.final_state && p1 == s.len && mcol < R.dc) {
        float* dst = R.final_state + ((int64_t)s.seq * g.heads + head) * matrix;
#pragma unroll
        for (int i = 0; i < G::DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * i + seq_crow(r) + 4 * h;
                if (row < R.da) dst[(uint32_t)(row * R.dc + mcol)] = m[i][r];
            }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// The recurrence for one token: S' = l S + k v^T, o = scale q S'.  Bound by reading and writing the fp32 state once (8 d_k d_v bytes a head); everything else is
// 0.4 % of that.  A thread owns four columns of every RP-th row; eight rows are in flight per thread; the rows' partial sums of o meet in LDS.  Heads of
// small batches are cut into column slices so that the few states spread over more CUs.
// ------------------------------------------------------------------------------------------------------------------------------
struct DecayStepArgs {
    const bf16_t *q, *k, *v;
    bf16_t* out;
    const float *state, *log_decay;
    float* new_state;
    int heads, dk, dv, slice;
    int64_t q_b, q_h, k_b, k_h, v_b, v_h;
    float scale;
};
__global__ void __launch_bounds__(256) decay_step_kernel(const DecayStepArgs a) {
    __shared__ float sq[128], sk[128];
    __shared__ __attribute__((aligned(16))) float so[256 * 4];
    const int tid = threadIdx.x, head = (int)blockIdx.x % a.heads;
    const int64_t b = blockIdx.x / a.heads;
    const int c0 = (int)blockIdx.y * a.slice, vec = min(a.slice, a.dv - c0) / 4, rp = 256 / vec, r0 = tid / vec, c = c0 + (tid % vec) * 4;
    if (tid < a.dk) {
        sq[tid] = bf16_to_f32(a.q[b * a.q_b + head * a.q_h + tid]);
        sk[tid] = bf16_to_f32(a.k[b * a.k_b + head * a.k_h + tid]);
    }
    const bool on = r0 < rp;
    const int64_t at = ((int64_t)b * a.heads + head) * a.dk * a.dv + c;
    const float* src = a.state + at;
    float* dst = a.new_state + at;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
    if (on) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(a.v + b * a.v_b + head * a.v_h + c);
        v = f32x4_t{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
    }
    const float l = __expf(a.log_decay[head]);
    __syncthreads();
    if (on)
        for (int base = r0; base < a.dk; base += 8 * rp) {
            f32x4_t x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const f32x4_t*>(src + (uint32_t)(min(base + i * rp, a.dk - 1) * a.dv));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = base + i * rp;
                const float kk = sk[min(row, 127)], qq = row < a.dk ? sq[min(row, 127)] : 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][e] = __builtin_fmaf(x[i][e], l, kk * v[e]);
                    o[e] = row < a.dk ? __builtin_fmaf(qq, x[i][e], o[e]) : o[e];
                }
                if (row < a.dk) *reinterpret_cast<f32x4_t*>(dst + (uint32_t)(row * a.dv)) = x[i];
            }
        }
    *reinterpret_cast<f32x4_t*>(so + tid * 4) = o;
    __syncthreads();
    if (tid < vec) {
        for (int j = 1; j < rp; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += so[(j * vec + tid) * 4 + e];
        const u32x2_t w = {pack_bf16x2(o[0] * a.scale, o[1] * a.scale), pack_bf16x2(o[2] * a.scale, o[3] * a.scale)};
        *reinterpret_cast<u32x2_t*>(a.out + (b * a.heads + head) * a.dv + c) = w;
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// C entry points
// ------------------------------------------------------------------------------------------------------------------------------
// tokens per segment: about 1024 blocks over the chip, but not under 256 tokens (a segment's state costs as much traffic as 128 / 256 tokens of it at head
// width 64 / 128) and not over 4096
static int decay_segment(int64_t rows, int heads) {
    int seg = 256;
    while (seg < 4096 && rows * heads / seg > 1024) seg *= 2;
    return seg;
}

extern "C" int64_t genie_decay_attention_ws_floats(int nseq, int rows, int heads, int dk, int dv) {
    if (nseq <= 0 || rows <= 0 || heads <= 0 || dk <= 0 || dv <= 0) return 0;
    const int seg = decay_segment(rows, heads);
    return rows <= seg ? 0 : (int64_t)(rows / seg + nseq + 1) * heads * dk * dv;
}

static int decay_check(const char* what, const DecayArgs& g) {
    GENIE_CHECK_ARG(g.cu && g.log_decay, "%s: null pointer", what);
    GENIE_CHECK_ARG(g.nseq >= 0 && g.rows > 0 && g.rows <= (1 << 30) && g.heads > 0, "%s: bad sizes (sequences %d, rows %d, heads %d)", what, g.nseq, g.rows, g.heads);
    GENIE_CHECK_ARG(g.scale == g.scale && g.scale < 1e30f && g.scale > -1e30f, "%s: scale must be finite", what);
    return GENIE_OK;
}
static int decay_check_role(const char* what, const DecayRole& r) {
    GENIE_CHECK_ARG(r.a && r.b && r.c && r.y, "%s: null pointer", what);
    GENIE_CHECK_ARG(r.da > 0 && r.da % 8 == 0 && r.da <= 128 && r.dc > 0 && r.dc % 8 == 0 && r.dc <= 128,
                    "%s: head widths %d, %d (multiples of 8 up to 128 are supported)", what, r.da, r.dc);
    const int64_t s[6] = {r.a_row, r.a_head, r.b_row, r.b_head, r.c_row, r.c_head};
    const int d[3] = {r.da, r.da, r.dc};
    for (int i = 0; i < 6; ++i) GENIE_CHECK_ARG(s[i] >= 0 && s[i] % 8 == 0, "%s: strides must be multiples of 8 elements", what);
    for (int i = 0; i < 3; ++i)
        GENIE_CHECK_ARG(s[2 * i] >= d[i] && s[2 * i] < (1 << 21), "%s: row stride %lld (the head width up to 2^21 elements is supported)", what, (long long)s[2 * i]);
    return GENIE_OK;
}

template <int DH>
static int decay_run(const DecayArgs& g, int roles, bool build_states, bool empties, void* stream) {
    const int NT = DecayGeo<DH>::NT;
    const int64_t blocks = (int64_t)g.nslots * g.heads;
    GENIE_CHECK_ARG(blocks + (int64_t)g.nseq * g.heads < (1ll << 31), "decay attention: too many blocks");
    if (build_states && g.rows > g.seg && g.nseq > 0) {
        hipLaunchKernelGGL(decay_state_kernel<DH>, dim3((unsigned)blocks), dim3(NT), 0, (hipStream_t)stream, g);
        GENIE_CHECK_LAUNCH();
        const int matrix = g.r[0].da * g.r[0].dc;
        hipLaunchKernelGGL(decay_scan_kernel, dim3((unsigned)(g.nseq * g.heads), (unsigned)((matrix + 1023) / 1024)), dim3(256), 0, (hipStream_t)stream, g, matrix);
        GENIE_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(decay_sweep_kernel<DH>, dim3((unsigned)(blocks + (empties ? (int64_t)g.nseq * g.heads : 0)), roles), dim3(NT), 0, (hipStream_t)stream, g);
    GENIE_CHECK_LAUNCH();
    return GENIE_OK;
}
static int decay_run_any(const DecayArgs& g, int roles, bool build_states, bool empties, void* stream) {
    const int d = g.r[0].da > g.r[0].dc ? g.r[0].da : g.r[0].dc;
    if (d <= 32) return decay_run<32>(g, roles, build_states, empties, stream);
    if (d <= 64) return decay_run<64>(g, roles, build_states, empties, stream);
    if (d <= 96) return decay_run<96>(g, roles, build_states, empties, stream);
    return decay_run<128>(g, roles, build_states, empties, stream);
}

extern "C" int genie_decay_attention_fwd(const void* q, const void* k, const void* v, const float* log_decay, const int32_t* cu, const float* initial_state, void* out,
                                         float* final_state, float* seg_ws, int64_t seg_ws_floats, int nseq, int rows, int heads, int dk, int dv,
                                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, float scale, void* stream) {
    const char* what = "genie_decay_attention_fwd";
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides, "%s: null strides", what);
    DecayArgs g = {};
    g.cu = cu; g.log_decay = log_decay; g.nseq = nseq; g.rows = rows; g.heads = heads; g.scale = scale;
    int rc = decay_check(what, g);
    if (rc != GENIE_OK) return rc;
    g.seg = decay_segment(rows, heads);
    g.nslots = rows / g.seg + nseq + 1;
    DecayRole& r = g.r[0];
    r.a = (const bf16_t*)q; r.b = (const bf16_t*)k; r.c = (const bf16_t*)v; r.y = (bf16_t*)out;
    r.a_row = q_strides[0]; r.a_head = q_strides[1]; r.b_row = k_strides[0]; r.b_head = k_strides[1]; r.c_row = v_strides[0]; r.c_head = v_strides[1];
    r.da = dk; r.dc = dv; r.m_a = dv; r.m_c = 1; r.seq_state = initial_state; r.seg_state = seg_ws; r.final_state = final_state;
    rc = decay_check_role(what, r);
    if (rc != GENIE_OK) return rc;
    GENIE_CHECK_ARG(seg_ws_floats >= genie_decay_attention_ws_floats(nseq, rows, heads, dk, dv) && (seg_ws || rows <= g.seg), "%s: workspace too small", what);
    return decay_run_any(g, 1, true, final_state != nullptr, stream);
}

extern "C" int genie_decay_attention_bwd(const void* q, const void* k, const void* v, const void* dout, const float* log_decay, const int32_t* cu,
                                         const float* initial_state, float* seg_ws, float* rev_ws, int64_t ws_floats, void* dq, void* dk_out, void* dv_out, int nseq,
                                         int rows, int heads, int dk, int dv, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                         const int64_t* dout_strides, float scale, void* stream) {
    const char* what = "genie_decay_attention_bwd";
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides && dout_strides, "%s: null strides", what);
    DecayArgs g = {};
    g.cu = cu; g.log_decay = log_decay; g.nseq = nseq; g.rows = rows; g.heads = heads; g.scale = scale;
    int rc = decay_check(what, g);
    if (rc != GENIE_OK) return rc;
    g.seg = decay_segment(rows, heads);
    g.nslots = rows / g.seg + nseq + 1;
    // role 0 is the one whose states are built here (reverse, from q and do): dv.  Role 1 uses their transposes: dk.  Role 2 uses the forward's: dq.
    DecayRole &rv = g.r[0], &rk = g.r[1], &rq = g.r[2];
    rv.a = (const bf16_t*)k; rv.b = (const bf16_t*)q; rv.c = (const bf16_t*)dout; rv.y = (bf16_t*)dv_out;
    rv.a_row = k_strides[0]; rv.a_head = k_strides[1]; rv.b_row = q_strides[0]; rv.b_head = q_strides[1]; rv.c_row = dout_strides[0]; rv.c_head = dout_strides[1];
    rv.da = dk; rv.dc = dv; rv.reverse = 1; rv.m_a = dv; rv.m_c = 1; rv.seg_state = rev_ws;
    rk.a = (const bf16_t*)v; rk.b = (const bf16_t*)dout; rk.c = (const bf16_t*)q; rk.y = (bf16_t*)dk_out;
    rk.a_row = v_strides[0]; rk.a_head = v_strides[1]; rk.b_row = dout_strides[0]; rk.b_head = dout_strides[1]; rk.c_row = q_strides[0]; rk.c_head = q_strides[1];
    rk.da = dv; rk.dc = dk; rk.reverse = 1; rk.m_a = 1; rk.m_c = dv; rk.seg_state = rev_ws;
    rq.a = (const bf16_t*)dout; rq.b = (const bf16_t*)v; rq.c = (const bf16_t*)k; rq.y = (bf16_t*)dq;
    rq.a_row = dout_strides[0]; rq.a_head = dout_strides[1]; rq.b_row = v_strides[0]; rq.b_head = v_strides[1]; rq.c_row = k_strides[0]; rq.c_head = k_strides[1];
    rq.da = dv; rq.dc = dk; rq.reverse = 0; rq.m_a = 1; rq.m_c = dv; rq.seq_state = initial_state; rq.seg_state = seg_ws;
    for (int i = 0; i < 3; ++i) {
        rc = decay_check_role(what, g.r[i]);
        if (rc != GENIE_OK) return rc;
    }
    GENIE_CHECK_ARG(ws_floats >= genie_decay_attention_ws_floats(nseq, rows, heads, dk, dv) && ((seg_ws && rev_ws) || rows <= g.seg), "%s: workspace too small", what);
    return decay_run_any(g, 3, true, false, stream);
}

extern "C" int genie_decay_attention_step(const void* q, const void* k, const void* v, const float* log_decay, const float* state, float* new_state, void* out, int batch,
                                          int heads, int dk, int dv, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, float scale,
                                          void* stream) {
    const char* what = "genie_decay_attention_step";
    GENIE_CHECK_ARG(q && k && v && log_decay && state && new_state && out && q_strides && k_strides && v_strides, "%s: null pointer", what);
    GENIE_CHECK_ARG(batch > 0 && heads > 0 && (int64_t)batch * heads < (1ll << 31), "%s: bad sizes (batch %d, heads %d)", what, batch, heads);
    GENIE_CHECK_ARG(dk > 0 && dk % 8 == 0 && dk <= 128 && dv > 0 && dv % 8 == 0 && dv <= 128, "%s: head widths %d, %d (multiples of 8 up to 128 are supported)", what, dk, dv);
    GENIE_CHECK_ARG(scale == scale && scale < 1e30f && scale > -1e30f, "%s: scale must be finite", what);
    DecayStepArgs a = {};
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.out = (bf16_t*)out; a.state = state; a.new_state = new_state; a.log_decay = log_decay;
    a.heads = heads; a.dk = dk; a.dv = dv; a.scale = scale;
    a.q_b = q_strides[0]; a.q_h = q_strides[1]; a.k_b = k_strides[0]; a.k_h = k_strides[1]; a.v_b = v_strides[0]; a.v_h = v_strides[1];
    const int64_t s[6] = {a.q_b, a.q_h, a.k_b, a.k_h, a.v_b, a.v_h};
    for (int i = 0; i < 6; ++i) GENIE_CHECK_ARG(s[i] >= 0 && s[i] % 4 == 0, "%s: strides must be multiples of 4 elements", what);
    a.slice = (int64_t)batch * heads < 256 && dv > 32 ? 32 : dv;
    hipLaunchKernelGGL(decay_step_kernel, dim3((unsigned)(batch * heads), (unsigned)((dv + a.slice - 1) / a.slice)), dim3(256), 0, (hipStream_t)stream, a);
    GENIE_CHECK_LAUNCH();
    return GENIE_OK;
}
