// Device helpers shared by the kernels that walk PACKED sequences (packed_attention.hip, decay_attention.hip) or a cache (cached_attention.hip):
// the slot -> (sequence, tile) search, range-checked loads, the transposing LDS read as a builtin.
#pragma once
#include "attn_common.h"

// ------------------------------------------------------------------------------------------------------------------------------
// Work list of packed sequences without a host round trip.  Sequence s owns the slots from f(s) = cu[s] / TILE + s on: f is strictly
// increasing and f(s + 1) - f(s) >= ceil(len_s / TILE), so every tile has a slot, at most nseq + 1 slots stay empty, and the number of slots
// is known from the sizes alone: rows / TILE + nseq + 1.  The last, virtual sequence (index nseq) holds the rows behind the last real one.
// cu is device memory nobody has checked: entries are clamped to [0, rows], so that wrong ones cost wrong results, never an access out of bounds.
// ------------------------------------------------------------------------------------------------------------------------------
struct SeqSlot { int seq, start, len, tile; };

__device__ __forceinline__ int seq_cu(const int32_t* cu, int s, int rows) { return s <= 0 ? 0 : min(max(cu[s], 0), rows); }

// The search is 64-way: one load and one ballot per level (one level up to 63 sequences), the same in every wave of the block.
template <int TILE>
__device__ __forceinline__ SeqSlot seq_find(const int32_t* cu, int nseq, int rows, int slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = nseq + 1;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int i = lane * step;
        const bool ok = i < n && seq_cu(cu, lo + i, rows) / TILE + lo + i <= slot;
        const int cnt = max(1, (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(ok)));
        lo += (cnt - 1) * step;
        n = min(step, n - (cnt - 1) * step);
    }
    SeqSlot r;
    r.seq = __builtin_amdgcn_readfirstlane(lo);
    r.start = __builtin_amdgcn_readfirstlane(seq_cu(cu, r.seq, rows));
    const int end = r.seq < nseq ? __builtin_amdgcn_readfirstlane(seq_cu(cu, r.seq + 1, rows)) : rows;
    r.len = max(0, end - r.start);
    r.tile = slot - (r.start / TILE + r.seq);
    return r;
}

// The same list in descending order of the rows of its sequence behind (or, FIRST, in front of) a tile, which is what a causal tile costs: the longest blocks start
// first, over all sequences.  Up to 63 sequences a lane holds one sequence's tile count n; C(u) = sum of max(0, n - u) tiles have u tiles or more on that side.
// The lanes try 63 values of u at a time (one level up to 63 tiles, two up to 3969, ..), a ballot finds the u of rank `slot`, another its sequence.  More
// sequences: the order of the slots above, from the end (FIRST: from the start).
template <int TILE, bool FIRST>
__device__ __forceinline__ SeqSlot seq_find_longest(const int32_t* cu, int nseq, int rows, int slot, int nslots) {
    if (nseq > 63) return seq_find<TILE>(cu, nseq, rows, FIRST ? slot : nslots - 1 - slot);
    const int lane = threadIdx.x & 63;
    const int start = seq_cu(cu, min(lane, nseq), rows), next = seq_cu(cu, min(lane + 1, nseq), rows);
    const int n = (max(0, next - start) + TILE - 1) / TILE;
    SeqSlot r;
    int lo = 0, range = rows / TILE + 2, above = 0;                             // C(lo) > slot; above: C(lo + 1) in the end
    do {
        const int step = (range + 62) / 63, u = lo + lane * step;
        int c = 0;
        for (int q = 0; q < nseq; ++q) c += max(0, __builtin_amdgcn_readlane(n, q) - u);
        if (lo == 0) {
            const int total = __builtin_amdgcn_readfirstlane(c);
            if (slot >= total) {                                                // the rows behind the last sequence
                r.seq = nseq;
                r.start = __builtin_amdgcn_readlane(start, nseq);
                r.len = rows - r.start;
                r.tile = slot - total;
                return r;
            }
        }
        const int cnt = max(1, (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(c > slot)));      // C descends: the first cnt lanes (lane 63 is past the end)
        lo += (cnt - 1) * step;
        above = __builtin_amdgcn_readlane(c, min(cnt, 63));
        range = step;
    } while (range > 1);
    // tiles with exactly lo behind them: one of every sequence with n > lo, after the C(lo + 1) longer ones
    uint64_t who = __builtin_amdgcn_ballot_w64(n > lo);
    for (int k = slot - above; k > 0; --k) who &= who - 1;
    r.seq = who ? (int)__builtin_ctzll(who) : 0;
    r.start = __builtin_amdgcn_readlane(start, r.seq);
    r.len = max(0, __builtin_amdgcn_readlane(next, r.seq) - r.start);
    r.tile = FIRST ? (r.len + TILE - 1) / TILE - 1 - lo : lo;
    return r;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Range-checked 16-B load: lanes whose offset reaches past `bytes_left` get zeros.  Offsets are inside one tile (the base moves in 64 bits), and the
// host refuses row strides whose tile does not fit 2^29 bytes.  SEQ_OOB marks a lane that never has data (columns behind the head's width).
// ------------------------------------------------------------------------------------------------------------------------------
#define SEQ_OOB 0x7ff00000u
// STREAM: non-temporal, for data that is read once.
template <bool STREAM = false>
__device__ __forceinline__ u32x4_t seq_load16(const void* base, int bytes_left, uint32_t voff) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes_left, 0x00020000);
    return __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, STREAM ? 2 : 0);
}
// the same load with its destination in LDS: lane l's 16 B go to lds + 16 l (lds is wave-uniform)
__device__ __forceinline__ void seq_dma16(const void* base, int bytes_left, char* lds, uint32_t voff) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes_left, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, LDS_PTR(lds), 16, voff, 0u, 0, 0);
}
// bytes a tile of at most 128 rows may read from its first row on, when `rows` rows remain (row strides are under 2^22 bytes: 32 bits hold it)
__device__ __forceinline__ int seq_bytes_left(int rows, int64_t stride_bytes, int dim) {
    return rows <= 0 ? 0 : (min(rows, 128) - 1) * (int)stride_bytes + dim * 2;
}

// ds_read_b64_tr_b16: in each group of 16 lanes, lane i names 4 consecutive 16-bit values of row i / 4 (columns 4 (i % 4) ...) and receives column i of the
// four rows.  The builtin: the compiler tracks the wait itself, but waits for an LDS-DMA in flight as well.
typedef __attribute__((address_space(3))) bf16x4_t seq_lds_b16x4;
__device__ __forceinline__ bf16x4_t seq_tr16(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((seq_lds_b16x4*)p); }

// Four fragments by eight such reads and their wait in ONE asm block: for loops with an LDS-DMA in flight, where the compiler would wait for the DMA in front of the
// builtin.  a0, a1: LDS byte addresses of fragments 0 and 1 (lower and upper half each); OFF1: byte distance of fragments 2 and 3.
template <int OFF0, int OFF1>
__device__ __forceinline__ void seq_tr16x4(bf16x8_t (&f)[4], uint32_t a0lo, uint32_t a0hi, uint32_t a1lo, uint32_t a1hi) {
    bf16x4_t r0, r1, r2, r3, r4, r5, r6, r7;
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %10 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3), "=&v"(r4), "=&v"(r5), "=&v"(r6), "=&v"(r7)
                 : "v"(a0lo), "v"(a0hi), "v"(a1lo), "v"(a1hi), "n"(OFF0), "n"(OFF1)
                 : "memory");
    f[0] = __builtin_shufflevector(r0, r1, 0, 1, 2, 3, 4, 5, 6, 7);
    f[1] = __builtin_shufflevector(r2, r3, 0, 1, 2, 3, 4, 5, 6, 7);
    f[2] = __builtin_shufflevector(r4, r5, 0, 1, 2, 3, 4, 5, 6, 7);
    f[3] = __builtin_shufflevector(r6, r7, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ bf16x8_t seq_pack8(const float a0, const float a1, const float a2, const float a3, const float a4, const float a5, const float a6,
                                              const float a7) {
    const u32x4_t v = {pack_bf16x2(a0, a1), pack_bf16x2(a2, a3), pack_bf16x2(a4, a5), pack_bf16x2(a6, a7)};
    return __builtin_bit_cast(bf16x8_t, v);
}
// what rounding to bf16 left over of x, rounded in its turn: x = hi + rest within 2^-17 of x
__device__ __forceinline__ bf16x8_t seq_rest8(const float (&x)[8], bf16x8_t hi) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e] - bf16_to_f32((bf16_t)hi[e]);
    return seq_pack8(r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]);
}

// value of the partner lane (lane ^ 32) combined with this lane's.  Inline asm as in the other attention kernels: given two copies of one value the
// builtin is folded as if the swap were the identity; no memory is involved, `s_nop 1` covers the VALU-write -> permlane-read hazard.
__device__ __forceinline__ void seq_swap32(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float seq_xmax32(float x) { float a = x, b = x; seq_swap32(a, b); return fmaxf(a, b); }
__device__ __forceinline__ float seq_xsum32(float x) { float a = x, b = x; seq_swap32(a, b); return a + b; }

// row of accumulator register r in the 32 x 32 MFMA result layout (column = lane & 31), h = lane >> 5
__device__ __forceinline__ constexpr int seq_crow(int r) { return (r & 3) + 8 * (r >> 2); }
