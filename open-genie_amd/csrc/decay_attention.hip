// Linear attention with a decay for each head over packed sequences (chunked form, forward and backward) and its recurrence for single tokens.
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   l = exp(log_decay[head])                (S: d_k x d_v, fp32)
//
// The forward and the three gradients are ONE form,  y_t = scale sum_{s <= t} l^(t-s) (a_t . b_s) c_s :
//   o = form(q, k, v)   dq = form(do, v, k)   and, run from the sequence's end,   dv = form(k, q, do)   dk = form(v, do, q)
// Segments of 256 tokens:  y_t = l^(t+1) a_t M + sum over the segment's own s <= t,  M = the state in front of the segment (for dq the transpose of the
// forward's, for dk that of dv's).  Three kernels:
//   state: what each segment adds, sum_s l^(n-1-s) b_s c_s^T          -- reads B and C once; parallel over segments, 64 tokens at a time
//   scan:  the states in front of the segments, elementwise in fp32    -- stored as the bf16 operand that the products take
//   out:   all rows at once, a wave owns 32: its product with M, then the segment's keys up to its diagonal, as softmax attention without the softmax
// A single walk through each sequence that keeps M in registers would read everything once, but has only (sequences x heads) blocks and
// a chain of dependent products per 64 tokens.  256 tokens balance the quadratic part (2.5 tiles of 64 keys a row) against the states
// (at head width 128 an fp32 matrix is as large as 128 tokens of q, k, v and o).
// All powers have exponents >= 0 (strong decays underflow to 0, nothing overflows).
//
// Roundings to bf16: the scores and M as matrix operands of an output that is itself rounded to bf16 (up to 256 rows: as two values each, 2^-17 left).  The states themselves are fp32 and so is what goes into them:
// the state update's decayed operand l^(n-1-s) c_s enters as a sum of three bf16 values (2^-24 left: fp32).  The backward's states, which only become
// operands of gradients, take two (2^-16, far under the operand's own 2^-8).
//
// Bound by memory and its latency.  Seven sequences of 16092 tokens, 16 heads of width 128 (66 MB a tensor): state 47 us, scan 18, outputs 68 forward and 156 for the three
// gradients; one prompt of 32768 tokens, 8 heads of width 64 (34 MB a tensor): 21 + 8 + 36 us, about 250 MB moved at 3.8 TB/s (a large copy: 4.9).  All on cold inputs.
#include "packed_common.h"

#define DECAY_SEG 256

struct DecayRole {
    const bf16_t *a, *b, *c;
    bf16_t* y;                                   // [rows][heads][dc]
    int64_t a_row, a_head, b_row, b_head, c_row, c_head;
    int da, dc, reverse, m_rows_a;               // m_rows_a: the stored states' rows are a's columns (else c's): the transposed use
    float* local;                                // [slot][heads][dc][da] fp32: what each segment adds
    bf16_t* states;                              // [slot][heads][dc][da] (m_rows_a: [da][dc]): state in front of each segment, or NULL
    int64_t rest;                                // elements from a state to what its rounding left over (0: not kept)
    const float* initial;                        // [nseq][heads][da][dc]: state in front of each sequence, or NULL
    float* final_state;                          // [nseq][heads][da][dc], or NULL
};
struct DecayArgs {
    DecayRole r[3];
    const int32_t* cu;
    const float* log_decay;
    int nseq, rows, heads, roles;
    float scale;
};

template <int DH>
struct DecayGeo {
    static constexpr int NW = DH / 32, NT = 64 * NW, CPR = DH / 8, PITCH = DH <= 64 ? 128 : 256, SW = PITCH / 16, KS = DH / 16, DT = DH / 32;
    static constexpr int TILE = 64 * PITCH, PIECES = 4;
};

// l^e for e >= 0 (l = 0 included: l^0 = 1)
__device__ __forceinline__ float decay_pow(float log2_l, int e) { return e == 0 ? 1.f : __builtin_amdgcn_exp2f(log2_l * (float)e); }

// One 64-token tile of a matrix from memory into registers and on to LDS.  A chunk with nv < 64 tokens (a segment's last) sits in the tile's LAST rows, so that
// the weights towards the chunk's end, l^(63-s), hold for it too; the rows in front of it read zeros: their offsets wrap past any range (forward) or lie
// behind the last token (reverse, where row i of the tile is the token 63 - i rows up in memory).
// A thread's four pieces are 16 rows apart in one column chunk (the swizzle's keys use row bits 0..3: one LDS address and constant offsets).
template <int DH>
struct DecayTile {
    using G = DecayGeo<DH>;
    static_assert(G::NT / G::CPR == 16 && G::NT % G::CPR == 0, "pieces are 16 rows apart");
    uint32_t off, lds;
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
        step = c * 8 < dim ? (int)(reverse ? -32 * stride : 32 * stride) : 0;
        lds = packed_at<DH>(rr, c);
    }
    // the chunk of tokens p .. p + nv - 1 of the walk over a sequence of len tokens (reverse: counted from its end)
    __device__ __forceinline__ void load(int p, int nv, int len) {
        const bf16_t* t = base + (int64_t)(rev ? len - p - nv : p) * row;
        const int left = seq_bytes_left(nv, row * 2, dim);
        const uint32_t o = off - (rev ? 0u : (uint32_t)((64 - nv) * row * 2));
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) r[i] = seq_load16(t, left, o + (uint32_t)(i * step));
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < G::PIECES; ++i) *reinterpret_cast<u32x4_t*>(tile + lds + i * 16 * G::PITCH) = r[i];
    }
};

// What one segment adds to the state, M = sum_s l^(n-1-s) b_s c_s^T over its n tokens, stored transposed ([dc][da]); wave w owns columns 32 w .. of C.  A
// sequence's last segment is only needed where the final state is.  DIRECT: every sequence is one segment and starts from nothing: the sum is the final state.
template <int DH, int TERMS, bool DIRECT>
__device__ __forceinline__ void decay_state_block(const DecayArgs& g, int block, char* smem) {      // 64 (DH / 32) threads; smem: 2 TILE
    using G = DecayGeo<DH>;
    const DecayRole& R = g.r[0];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int head = block % g.heads, slot = block / g.heads;
    const SeqSlot s = seq_find<DECAY_SEG>(g.cu, g.nseq, g.rows, slot);
    const int p0 = s.tile * DECAY_SEG;
    if (s.seq == g.nseq || s.tile < 0 || p0 >= max(s.len, DIRECT ? 1 : 0)) return;      // (DIRECT: an empty sequence's state is written too)
    if (p0 + DECAY_SEG >= s.len && !R.final_state) return;
    const int p1 = min(s.len, p0 + DECAY_SEG);
    const float log2_l = g.log_decay[head] * 1.4426950408889634f;
    float fade[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) fade[r] = decay_pow(log2_l, 31 - (seq_crow(r) + 4 * h));
    const float p32 = decay_pow(log2_l, 32);
    PackedLane<DH> at;
    at.init(lane);
    DecayTile<DH> tb, tc;
    tb.init(tid, R.b + (int64_t)s.start * R.b_row + head * R.b_head, R.b_row, R.da, R.reverse);
    tc.init(tid, R.c + (int64_t)s.start * R.c_row + head * R.c_head, R.c_row, R.dc, R.reverse);
    f32x16_t m[G::DT];
#pragma unroll
    for (int i = 0; i < G::DT; ++i) m[i] = packed_splat(0.f);
    char *bt = smem, *ct = smem + G::TILE;
    // the chunk that does not fill a tile comes first: all others end where the next one begins
    int nv = (p1 - p0 + 63) % 64 + 1;
    if (p0 < p1) {
        tb.load(p0, nv, s.len);
        tc.load(p0, nv, s.len);
    }
    for (int p = p0; p < p1;) {
        tb.store(bt);
        tc.store(ct);
        __syncthreads();
        p += nv;
        nv = 64;
        if (p < p1) {
            tb.load(p, 64, s.len);
            tc.load(p, 64, s.len);
        }
        at.forget();
#pragma unroll
        for (int i = 0; i < G::DT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) m[i][r] *= p32 * p32;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const bf16x8_t cf = at.tr_frag(ct + ks * 16 * G::PITCH, wave);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = bf16_to_f32((bf16_t)cf[j]) * fade[8 * (ks & 1) + j];
                if (ks < 2) x[j] *= p32;
            }
            bf16x8_t part[TERMS];                                               // x = the sum of the parts
#pragma unroll
            for (int n = 0; n < TERMS; ++n) {
                const u32x4_t f = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
                part[n] = __builtin_bit_cast(bf16x8_t, f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[2 * j] -= __uint_as_float(f[j] << 16);
                    x[2 * j + 1] -= __uint_as_float(f[j] & 0xffff0000u);
                }
            }
#pragma unroll
            for (int i = 0; i < G::DT; ++i) {
                const bf16x8_t bf = at.tr_frag(bt + ks * 16 * G::PITCH, i);
#pragma unroll
                for (int n = TERMS - 1; n >= 0; --n) m[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(part[n], bf, m[i], 0, 0, 0);
            }
        }
        __syncthreads();
    }
    if (DIRECT) {                                                               // natural layout: four consecutive columns of a row per store
        float* dst = R.final_state + ((int64_t)s.seq * g.heads + head) * R.da * R.dc;
#pragma unroll
        for (int i = 0; i < G::DT; ++i) {
            const int row = 32 * i + (lane & 31);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = 32 * wave + 8 * q + 4 * h;
                if (row < R.da && col < R.dc)
                    *reinterpret_cast<f32x4_t*>(dst + (uint32_t)(row * R.dc + col)) = f32x4_t{m[i][4 * q], m[i][4 * q + 1], m[i][4 * q + 2], m[i][4 * q + 3]};
            }
        }
        return;
    }
    float* dst = R.local + ((int64_t)slot * g.heads + head) * R.da * R.dc;
#pragma unroll
    for (int i = 0; i < G::DT; ++i) {
        const int col = 32 * i + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = 32 * wave + seq_crow(r) + 4 * h;
            if (col < R.da && row < R.dc) dst[(uint32_t)(row * R.da + col)] = m[i][r];
        }
    }
}

template <int DH, int TERMS>
__global__ void __launch_bounds__(64 * (DH / 32), 2) decay_state_kernel(const DecayArgs g) {
    __shared__ __attribute__((aligned(16))) char smem[2 * DecayGeo<DH>::TILE];
    decay_state_block<DH, TERMS, false>(g, (int)blockIdx.x, smem);
}

// States in front of the segments: M_0 = initial or 0, M_{i+1} = l^256 M_i + local_i, elementwise in fp32; each M_i is stored rounded to bf16 as the operand that it
// becomes, the last sum is the final state.  A lane owns four elements, the block's NW waves take eight segments each: all loads of a step are in flight
// together, the waves' sums meet in LDS, and each wave walks its own eight from there.  128 segments of 8 heads of width 64: 16 waves 8.3 us, 4 waves 9.8, one wave walking all
// of them, eight loads ahead, 18 -- a chain of store and load latencies.  Up to 32 segments a sequence four waves do it in one step: 100 MB of 63 segments of 16 heads of
// width 128 in 18 us = 5.5 TB/s (what the state kernel just wrote is partly still in the last-level cache).
template <int NW>
__global__ void __launch_bounds__(64 * NW) decay_scan_kernel(const DecayArgs g) {
    __shared__ __attribute__((aligned(16))) f32x4_t part[2][NW][64];
    const DecayRole& R = g.r[0];
    const int seq = (int)blockIdx.x / g.heads, head = (int)blockIdx.x % g.heads, matrix = R.da * R.dc;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int e0 = ((int)blockIdx.y * 64 + lane) * 4, e = min(e0, matrix - 4);   // (lanes past the end repeat the last elements' work and store the same)
    const int start = seq_cu(g.cu, seq, g.rows), len = max(0, seq_cu(g.cu, seq + 1, g.rows) - start), nseg = (len + DECAY_SEG - 1) / DECAY_SEG;
    const float log2_l = g.log_decay[head] * 1.4426950408889634f, l = decay_pow(log2_l, DECAY_SEG);
    const int c = e / R.da, a = e % R.da;                                       // elements (a .. a + 3, c) of the states that go in and out
    const int64_t of_seq = ((int64_t)seq * g.heads + head) * matrix;
    f32x4_t m = {0.f, 0.f, 0.f, 0.f};
    if (R.initial) {
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = R.initial[of_seq + (a + j) * R.dc + c];
    }
    const int64_t step = (int64_t)g.heads * matrix, first = ((int64_t)(start / DECAY_SEG + seq) * g.heads + head) * matrix + e;
    const float* src = R.local + first;
    bf16_t* dst = R.states + first;
    const int full = nseg - 1;                                                  // segments whose sum is followed by another segment
    const float l8 = decay_pow(log2_l, 8 * DECAY_SEG);
    for (int base = 0, flip = 0; base < full; base += 8 * NW, flip ^= 1) {
        const int i0 = base + wave * 8, n = min(8, full - i0);
        f32x4_t x[8], sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) x[j] = *reinterpret_cast<const f32x4_t*>(src + (i0 + j) * step);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[q] = __builtin_fmaf(sum[q], l, x[j][q]);
        part[flip][wave][lane] = sum;
        __syncthreads();
        f32x4_t mine = m;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w == wave) mine = m;
            const int nw = min(8, full - base - w * 8);
            if (nw > 0) {
                const float f = nw == 8 ? l8 : decay_pow(log2_l, nw * DECAY_SEG);
                const f32x4_t s = part[flip][w][lane];
#pragma unroll
                for (int q = 0; q < 4; ++q) m[q] = __builtin_fmaf(m[q], f, s[q]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) {
                *reinterpret_cast<u32x2_t*>(dst + (i0 + j) * step) = u32x2_t{pack_bf16x2(mine[0], mine[1]), pack_bf16x2(mine[2], mine[3])};
#pragma unroll
                for (int q = 0; q < 4; ++q) mine[q] = __builtin_fmaf(mine[q], l, x[j][q]);
            }
    }
    if (wave != 0) return;
    if (nseg > 0) {
        const u32x2_t hi = {pack_bf16x2(m[0], m[1]), pack_bf16x2(m[2], m[3])};
        *reinterpret_cast<u32x2_t*>(dst + (nseg - 1) * step) = hi;
        if (R.rest)                                                              // (calls of one segment per sequence: m is the initial state)
            *reinterpret_cast<u32x2_t*>(dst + (nseg - 1) * step + R.rest) =
                u32x2_t{pack_bf16x2(m[0] - __uint_as_float(hi[0] << 16), m[1] - __uint_as_float(hi[0] & 0xffff0000u)),
                        pack_bf16x2(m[2] - __uint_as_float(hi[1] << 16), m[3] - __uint_as_float(hi[1] & 0xffff0000u))};
    }
    if (!R.final_state) return;
    if (nseg > 0) {
        const f32x4_t last = *reinterpret_cast<const f32x4_t*>(src + (nseg - 1) * step);
        const float ln = decay_pow(log2_l, len - (nseg - 1) * DECAY_SEG);
#pragma unroll
        for (int q = 0; q < 4; ++q) m[q] = __builtin_fmaf(m[q], ln, last[q]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) R.final_state[of_seq + (a + j) * R.dc + c] = m[j];
}

// 32 rows straight into LDS, as PackedDma, for tokens walked in either direction (last >= 0: row i is token last - i from the base; rows behind the walk's end wrap
// past any range).
template <int DH>
struct DecayDma {
    using G = PackedGeo<DH>;
    static constexpr int SLABS = 32 * G::PITCH / 1024 / 4, ROWS = 1024 / G::PITCH;
    int row0, slot;
    __device__ __forceinline__ void init(int wave, int lane) { row0 = wave * SLABS * ROWS + lane / G::SW; slot = lane % G::SW; }
    __device__ __forceinline__ void load(int wave, char* tile, const bf16_t* base, int64_t stride, int rows, int dim, int last) {
        asm volatile("" : "+v"(row0), "+v"(slot));                              // (offsets are formed anew: registers are short)
        const int left = seq_bytes_left(rows, stride * 2, dim);
        const uint32_t pitch = (uint32_t)(stride * 2);
#pragma unroll
        for (int i = 0; i < SLABS; ++i) {
            const int row = row0 + i * ROWS, c = attn_swz<G::SW>(row, slot);
            const uint32_t o = (uint32_t)(last >= 0 ? last - row : row) * pitch + c * 16;
            seq_dma16(base, left, tile + (wave * SLABS + i) * 1024, c * 8 < dim ? o : SEQ_OOB);
        }
    }
};

// acc[d] += (transposed 32-row tile, columns 32 d ..) x p, d = 0 ..: the reads and their wait in asm blocks where two columns make one (the loads in flight stay there)
template <int DH>
__device__ __forceinline__ void decay_tr_product(f32x16_t (&acc)[PackedGeo<DH>::DT], const PackedLane<DH>& at, const char* tile, const bf16x8_t (&p)[2]) {
    using G = PackedGeo<DH>;
    if constexpr (G::DT % 2 == 0) {
        const uint32_t base = attn_lds_offset(tile);
#pragma unroll
        for (int d = 0; d < G::DT; d += 2) {
            bf16x8_t f[4];
            seq_tr16x4<0, 16 * G::PITCH>(f, base + (at.tr0 ^ (uint32_t)(d * 64)), base + (at.tr1 ^ (uint32_t)(d * 64)), base + (at.tr0 ^ (uint32_t)(d * 64 + 64)),
                                         base + (at.tr1 ^ (uint32_t)(d * 64 + 64)));
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[d + e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[2 * s2 + e], p[s2], acc[d + e], 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int d = 0; d < G::DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.tr_frag(tile + s2 * 16 * G::PITCH, d), p[s2], acc[d], 0, 0, 0);
    }
}

// All outputs of one role: four waves of 32 rows; the state in front of the segment, then the segment's keys, 32 at a time, pass through a ring of three LDS stages,
// two ahead (counted waits).  A block is short -- 4 or 8 key tiles -- and lives on memory latency: stages of 32 keys and the fade table in LDS make three blocks
// fit a CU (48 KB, 168 registers) at head width 128.  (66 MB tensors, three gradients: stages of 64 keys and two blocks per CU 240 us, so 222 at the time.  The forward's 73 us then
// fell to 41 without the key tiles, to 68 without the state, to 60 without the last write: no part alone is the bound.)
template <int DH>
constexpr int decay_out_lds = 3 * 64 * PackedGeo<DH>::PITCH + 128;
template <int DH, bool REST>
__device__ __forceinline__ void decay_out_block(const DecayArgs& g, int block, char* smem) {
    using G = PackedGeo<DH>;
    constexpr int BM = 128, STAGE = 64 * G::PITCH, MINE = 2 * DecayDma<DH>::SLABS;      // MINE: loads of a wave per stage
    // heads fastest, then roles: the roles read the same tensors (and two of them the same tiles), and with a multiple of 8 heads those blocks share an XCD's L2
    const int head = block % g.heads, role = block / g.heads % g.roles, slot = block / g.heads / g.roles;
    const DecayRole& R = g.r[role];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const SeqSlot s = seq_find<BM>(g.cu, g.nseq, g.rows, slot);
    if (s.tile < 0 || s.tile * BM >= s.len) return;
    if (s.seq == g.nseq) {
        packed_zero_rows<BM, 256>(R.y, g.heads, R.dc, s, head);
        return;
    }
    const int rev = R.reverse, r0 = s.tile * BM, seg = r0 / DECAY_SEG, seg0 = seg * DECAY_SEG, end = min(s.len, r0 + BM);
    const int q0 = r0 + wave * 32, qi = q0 + (lane & 31);                        // rows in the order of the walk
    const float log2_l = g.log_decay[head] * 1.4426950408889634f;
    const bool carried = R.states && (seg > 0 || R.initial);                     // M is not zero
    const int tiles = (end - seg0 + 31) >> 5;

    const bf16_t* arow = R.a + (int64_t)(s.start + (rev ? s.len - 1 - qi : qi)) * R.a_row + head * R.a_head;
    const bf16_t* bp = R.b + (int64_t)s.start * R.b_row + head * R.b_head;
    const bf16_t* cp = R.c + (int64_t)s.start * R.c_row + head * R.c_head;
    DecayDma<DH> st;
    st.init(wave, lane);
    auto stage = [&](int t) { return smem + (t + 2) % 3 * STAGE; };
    auto load = [&](int t) {
        char* to = stage(t);
        const int p = seg0 + t * 32, nv = min(32, s.len - p), from = rev ? s.len - p - nv : p;
        st.load(wave, to, bp + (int64_t)from * R.b_row, R.b_row, nv, R.da, rev ? nv - 1 : -1);
        st.load(wave, to + STAGE / 2, cp + (int64_t)from * R.c_row, R.c_row, nv, R.dc, rev ? nv - 1 : -1);
    };
    bf16x8_t af[G::KS];                                                          // (in front of the tiles' loads: the counted waits below count what is younger)
    packed_row_frags<DH>(af, arow, qi < s.len, R.da);
    auto load_state = [&](int64_t rest) {                                        // into stages 0 and 1
        const int mr = R.m_rows_a ? R.da : R.dc, mc = R.m_rows_a ? R.dc : R.da;
        const bf16_t* m = R.states + ((int64_t)(s.start / DECAY_SEG + s.seq + seg) * g.heads + head) * mr * mc + rest;
#pragma unroll
        for (int i = 0; i < G::DT; ++i) st.load(wave, smem + i * 32 * G::PITCH, m + i * 32 * mc, mc, mr - i * 32, mc, -1);
    };
    if (carried) load_state(0);
    load(0);
    if (!carried && tiles > 1) load(1);
    PackedLane<DH> at;
    at.init(lane);
    float* fade = reinterpret_cast<float*>(smem + 3 * STAGE);                     // [h][r]: l^(31 - row r of a 32-row half)
    if (tid < 32) fade[tid] = decay_pow(log2_l, 31 - ((tid & 3) + 8 * (tid >> 2 & 3) + 4 * (tid >> 4)));
    f32x16_t y[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) y[d] = packed_splat(0.f);

    if (carried) {
        auto times_state = [&]() __attribute__((always_inline)) {                // y += a M
            if (!R.m_rows_a) {
#pragma unroll
                for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
                    for (int d = 0; d < G::DT; ++d) y[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.row_frag(smem + d * 32 * G::PITCH, ks), af[ks], y[d], 0, 0, 0);
            } else {
                // the transposing read delivers columns of a in the accumulator order, 4 h .. + 3 and 8 + 4 h .. + 3 of 16; af holds 8 h .. + 7: the lanes of a row trade halves
#pragma unroll
                for (int k2 = 0; k2 < G::KS; k2 += 2) {
                    bf16x8_t ap[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const u32x4_t f = __builtin_bit_cast(u32x4_t, af[k2 + e]);
                        const auto x = __builtin_amdgcn_permlane32_swap(f[0], f[2], false, false), z = __builtin_amdgcn_permlane32_swap(f[1], f[3], false, false);
                        ap[e] = __builtin_bit_cast(bf16x8_t, u32x4_t{x[0], z[0], x[1], z[1]});
                    }
                    decay_tr_product<DH>(y, at, smem + k2 * 16 * G::PITCH, ap);
                }
            }
        };
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MINE) : "memory");
        __syncthreads();
        times_state();
        if (REST && R.rest) {                                                    // few rows: the state with what its rounding left over
            __syncthreads();
            load_state(R.rest);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            times_state();
        }
        const float lead = decay_pow(log2_l, qi - seg0 + 1);
#pragma unroll
        for (int d = 0; d < G::DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) y[d][r] *= lead;
        if (tiles > 1) {
            __syncthreads();                                                     // everybody is done with the state
            load(1);
        }
    }
    for (int t = 0; t < tiles; ++t) {
        char* bt = stage(t);
        char* ct = bt + STAGE / 2;
        if (t + 1 < tiles) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MINE) : "memory");      // tile t has landed, t + 1 is in flight
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 2 < tiles) load(t + 2);
        const int k0 = seg0 + t * 32;
        if (k0 > q0) continue;                                                   // (wave-uniform) behind this wave's rows
        at.forget();
        f32x16_t x = packed_splat(0.f);
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(at.row_frag(bt, ks), af[ks], x, 0, 0, 0);
        if (k0 == q0) {                                                          // the diagonal: l^(t-s) for s <= t
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = (lane & 31) - (seq_crow(r) + 4 * h);
                x[r] = d >= 0 ? x[r] * decay_pow(log2_l, max(0, d)) : 0.f;
            }
        } else {                                                                 // l^(t-s) = l^(31 - s) l^(t + 1 + distance of the tiles - 32)
            const float f = decay_pow(log2_l, (lane & 31) + 1 + q0 - k0 - 32);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_t w = *reinterpret_cast<const f32x4_t*>(fade + 16 * h + 4 * q);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * q + e] *= w[e] * f;
            }
        }
        bf16x8_t pf[2];
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
            pf[s2] = seq_pack8(x[8 * s2], x[8 * s2 + 1], x[8 * s2 + 2], x[8 * s2 + 3], x[8 * s2 + 4], x[8 * s2 + 5], x[8 * s2 + 6], x[8 * s2 + 7]);
        if (REST) {
            bf16x8_t pr[2];
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const float p[8] = {x[8 * s2], x[8 * s2 + 1], x[8 * s2 + 2], x[8 * s2 + 3], x[8 * s2 + 4], x[8 * s2 + 5], x[8 * s2 + 6], x[8 * s2 + 7]};
                pr[s2] = seq_rest8(p, pf[s2]);
            }
            decay_tr_product<DH>(y, at, ct, pr);
        }
        decay_tr_product<DH>(y, at, ct, pf);
    }
    __syncthreads();
    if (q0 < s.len) {
        const int64_t pitch = (int64_t)g.heads * R.dc;
        packed_write_rows<DH>(smem + wave * 32 * G::PITCH, y, g.scale, R.y + ((int64_t)(s.start + (rev ? s.len - 1 - q0 : q0)) * g.heads + head) * R.dc,
                              rev ? -pitch : pitch, min(32, s.len - q0), R.dc);
    }
}
template <int DH>
__global__ void __launch_bounds__(256, DH <= 64 ? 4 : 3) decay_out_kernel(const DecayArgs g) {
    __shared__ __attribute__((aligned(16))) char smem[decay_out_lds<DH>];
    decay_out_block<DH, false>(g, (int)blockIdx.x, smem);
}
// Few rows: the weights and the state in front of a sequence with what their rounding left over, for the reason at packed_exact() (a 32768-token prompt would pay 38 us for 33).  The
// state's remainder costs a second product after its own loads: 168 rows behind initial states 9.3 us for 8.4 at width 64, 12.1 for 10.6 at 128.  Where every sequence is one
// segment and starts from nothing, the final states come from the launch's last blocks: three snippets of 168 tokens together 8 us instead of 7 + 7 in two launches.
template <int DH>
__global__ void __launch_bounds__(256) decay_few_kernel(const DecayArgs g, int out_blocks) {
    __shared__ __attribute__((aligned(16))) char smem[decay_out_lds<DH>];
    static_assert(decay_out_lds<DH> >= 2 * DecayGeo<DH>::TILE, "room for the state's tiles");
    const int block = (int)blockIdx.x - out_blocks;
    if (block < 0) decay_out_block<DH, true>(g, (int)blockIdx.x, smem);
    else if (threadIdx.x < DecayGeo<DH>::NT) decay_state_block<DH, 3, true>(g, block, smem);
}

// ------------------------------------------------------------------------------------------------------------------------------
// The recurrence for one token: S' = l S + k v^T, o = scale q S'.  Bound by reading and writing the fp32 state once (8 d_k d_v bytes a head); everything else is
// 0.4 % of that.  A thread owns four columns of every RP-th row; eight rows are in flight per thread; the rows' partial sums of o meet in LDS.  Non-temporal loads,
// ordinary stores.  4096 states of 128 x 128 (541 MB), call on cold states 102 us = 5.3 TB/s: both ordinary 104, both non-temporal 96, ordinary loads and non-temporal stores 104; where the last call's
// states are still in the last-level cache, kernel 81: both ordinary 103, both non-temporal 95.  Heads of
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
            for (int i = 0; i < 8; ++i) x[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(src + (uint32_t)(min(base + i * rp, a.dk - 1) * a.dv)));
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
// matrix elements of a call's segment states (one bf16 operand and one fp32 sum each); none where every sequence is one segment and starts from nothing.  Up to a
// segment of rows with initial states: twice as many, the second half for what the operands' rounding left over.
static bool decay_keeps_rest(int rows, bool initial) { return initial && rows <= DECAY_SEG; }
extern "C" int64_t genie_decay_attention_state_elems(int nseq, int rows, int heads, int dk, int dv, int has_initial) {
    if (nseq <= 0 || rows <= 0 || heads <= 0 || dk <= 0 || dv <= 0 || (rows <= DECAY_SEG && !has_initial)) return 0;
    return (int64_t)(rows / DECAY_SEG + nseq + 1) * heads * dk * dv * (decay_keeps_rest(rows, has_initial) ? 2 : 1);
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

// role 0's states, then all roles' outputs
template <int DH>
static int decay_run(const DecayArgs& g, void* stream) {
    const int64_t segs = (int64_t)(g.rows / DECAY_SEG + g.nseq + 1) * g.heads, blocks = (int64_t)(g.rows / 128 + g.nseq + 1) * g.heads * g.roles;
    GENIE_CHECK_ARG(segs + blocks < (1ll << 31), "decay attention: too many blocks");
    const DecayRole& r = g.r[0];
    if (g.nseq > 0 && r.local) {
        auto* kernel = g.roles == 1 ? decay_state_kernel<DH, 3> : decay_state_kernel<DH, 2>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)segs), dim3(DecayGeo<DH>::NT), 0, (hipStream_t)stream, g);
        GENIE_CHECK_LAUNCH();
        const dim3 grid((unsigned)(g.nseq * g.heads), (unsigned)((r.da * r.dc + 255) / 256));
        if (g.rows > 32ll * DECAY_SEG * g.nseq) hipLaunchKernelGGL((decay_scan_kernel<16>), grid, dim3(1024), 0, (hipStream_t)stream, g);
        else hipLaunchKernelGGL((decay_scan_kernel<4>), grid, dim3(256), 0, (hipStream_t)stream, g);
        GENIE_CHECK_LAUNCH();
    }
    const int64_t direct = r.local || !r.final_state ? 0 : segs;                 // (without `local` and more rows than a segment there is no sequence)
    if (g.rows <= DECAY_SEG) hipLaunchKernelGGL((decay_few_kernel<DH>), dim3((unsigned)(blocks + direct)), dim3(256), 0, (hipStream_t)stream, g, (int)blocks);
    else hipLaunchKernelGGL((decay_out_kernel<DH>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, g);
    GENIE_CHECK_LAUNCH();
    return GENIE_OK;
}
static int decay_run_any(const DecayArgs& g, void* stream) {
    const int d = g.r[0].da > g.r[0].dc ? g.r[0].da : g.r[0].dc;
    if (d <= 32) return decay_run<32>(g, stream);
    if (d <= 64) return decay_run<64>(g, stream);
    if (d <= 96) return decay_run<96>(g, stream);
    return decay_run<128>(g, stream);
}

extern "C" int genie_decay_attention_fwd(const void* q, const void* k, const void* v, const float* log_decay, const int32_t* cu, const float* initial_state, void* out,
                                         float* final_state, void* states, float* ws, int64_t state_elems, int nseq, int rows, int heads, int dk, int dv,
                                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, float scale, void* stream) {
    const char* what = "genie_decay_attention_fwd";
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides, "%s: null strides", what);
    DecayArgs g = {};
    g.cu = cu; g.log_decay = log_decay; g.nseq = nseq; g.rows = rows; g.heads = heads; g.scale = scale;
    int rc = decay_check(what, g);
    if (rc != GENIE_OK) return rc;
    DecayRole& r = g.r[0];
    r.a = (const bf16_t*)q; r.b = (const bf16_t*)k; r.c = (const bf16_t*)v; r.y = (bf16_t*)out;
    r.a_row = q_strides[0]; r.a_head = q_strides[1]; r.b_row = k_strides[0]; r.b_head = k_strides[1]; r.c_row = v_strides[0]; r.c_head = v_strides[1];
    r.da = dk; r.dc = dv; r.states = (bf16_t*)states; r.local = ws; r.initial = initial_state; r.final_state = final_state;
    rc = decay_check_role(what, r);
    if (rc != GENIE_OK) return rc;
    const int64_t need = genie_decay_attention_state_elems(nseq, rows, heads, dk, dv, initial_state != nullptr);
    GENIE_CHECK_ARG(state_elems >= need && (need == 0 || (states && ws)), "%s: workspace too small", what);
    if (need == 0) { r.states = nullptr; r.local = nullptr; }
    r.rest = decay_keeps_rest(rows, initial_state) ? need / 2 : 0;
    g.roles = 1;
    return decay_run_any(g, stream);
}

extern "C" int genie_decay_attention_bwd(const void* q, const void* k, const void* v, const void* dout, const float* log_decay, const int32_t* cu, int has_initial,
                                         const void* states, void* rev_states, float* ws, int64_t state_elems, void* dq, void* dk_out, void* dv_out, int nseq, int rows,
                                         int heads, int dk, int dv, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                         const int64_t* dout_strides, float scale, void* stream) {
    const char* what = "genie_decay_attention_bwd";
    GENIE_CHECK_ARG(q_strides && k_strides && v_strides && dout_strides, "%s: null strides", what);
    DecayArgs g = {};
    g.cu = cu; g.log_decay = log_decay; g.nseq = nseq; g.rows = rows; g.heads = heads; g.scale = scale;
    int rc = decay_check(what, g);
    if (rc != GENIE_OK) return rc;
    // role 0 is the one whose states are built here (from the end, of q and do): dv.  Role 1 uses their transposes: dk.  Role 2 those of the forward's: dq.
    DecayRole &rv = g.r[0], &rk = g.r[1], &rq = g.r[2];
    rv.a = (const bf16_t*)k; rv.b = (const bf16_t*)q; rv.c = (const bf16_t*)dout; rv.y = (bf16_t*)dv_out;
    rv.a_row = k_strides[0]; rv.a_head = k_strides[1]; rv.b_row = q_strides[0]; rv.b_head = q_strides[1]; rv.c_row = dout_strides[0]; rv.c_head = dout_strides[1];
    rv.da = dk; rv.dc = dv; rv.reverse = 1;
    rk.a = (const bf16_t*)v; rk.b = (const bf16_t*)dout; rk.c = (const bf16_t*)q; rk.y = (bf16_t*)dk_out;
    rk.a_row = v_strides[0]; rk.a_head = v_strides[1]; rk.b_row = dout_strides[0]; rk.b_head = dout_strides[1]; rk.c_row = q_strides[0]; rk.c_head = q_strides[1];
    rk.da = dv; rk.dc = dk; rk.reverse = 1; rk.m_rows_a = 1;
    rq.a = (const bf16_t*)dout; rq.b = (const bf16_t*)v; rq.c = (const bf16_t*)k; rq.y = (bf16_t*)dq;
    rq.a_row = dout_strides[0]; rq.a_head = dout_strides[1]; rq.b_row = v_strides[0]; rq.b_head = v_strides[1]; rq.c_row = k_strides[0]; rq.c_head = k_strides[1];
    rq.da = dv; rq.dc = dk; rq.m_rows_a = 1; rq.states = (bf16_t*)const_cast<void*>(states);
    rq.initial = has_initial ? log_decay : nullptr;                             // (only asked whether it is there: the state itself is in `states`)
    for (int i = 0; i < 3; ++i) {
        rc = decay_check_role(what, g.r[i]);
        if (rc != GENIE_OK) return rc;
    }
    const int64_t need = genie_decay_attention_state_elems(nseq, rows, heads, dk, dv, 0);
    GENIE_CHECK_ARG(state_elems >= need && (need == 0 || (states && rev_states && ws)) && (!has_initial || states), "%s: workspace too small", what);
    if (need > 0) { rv.states = rk.states = (bf16_t*)rev_states; rv.local = ws; }
    rq.rest = decay_keeps_rest(rows, has_initial) ? genie_decay_attention_state_elems(nseq, rows, heads, dk, dv, 1) / 2 : 0;
    g.roles = 3;
    return decay_run_any(g, stream);
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
