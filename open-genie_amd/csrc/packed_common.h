// Shared by the kernels of packed causal attention (packed_attention.hip, packed_attention_dkv.hip): arguments, LDS layout, staging, epilogue.
#pragma once
#include "seq_common.h"
#include "genie_hip.h"

struct PackedArgs {
    const bf16_t *q, *k, *v, *o, *dout;
    bf16_t *out, *out_lo, *dq, *dk, *dv;      // out_lo: what the rounding of out left over, bf16, for rowsum(dO o O) (or NULL)
    float* lse;                    // [Hq][rows_q]  log-sum-exp of the scaled scores, -inf where a row sees nothing
    float* delta;                  // [Hq][rows_q]  rowsum(dO o O), written by the dQ kernel for the dK / dV kernel
    float* part;                   // [nsplit][dK, dV][rows_k][Hkv][dim] where a key tile's rows are split over blocks
    int nsplit;
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

// Lane offsets of the fragment reads.  Every other offset is one of these with constant bits flipped: the swizzle is an exclusive-or of the chunk with a key of row
// bits 0..3, so chunk step ks of a row is rows ^ 32 ks and column step d of a transposing read is tr ^ 64 d; 16 rows further is a constant.  Three
// registers instead of two dozen, one v_xad per read: the dK / dV kernel has none to spare.
//   rows: row lane & 31, chunk h (operand fragments of the tile itself)
//   tr0, tr1: rows 4 h + 0..3 and 8 + 4 h + 0..3 of a 16-row step, columns lane & 31 (the two transposing reads that make a fragment of the transposed tile)
template <int DH>
struct PackedLane {
    uint32_t rows, tr0, tr1;
    __device__ __forceinline__ void init(int lane) {
        const int g16 = lane >> 4, r0 = 4 * (g16 >> 1) + ((lane >> 2) & 3), col = 16 * (g16 & 1) + 4 * (lane & 3);
        rows = packed_at<DH>(lane & 31, lane >> 5);
        tr0 = packed_at<DH>(r0, col >> 3) + (col & 7) * 2;
        tr1 = packed_at<DH>(r0 + 8, col >> 3) + (col & 7) * 2;
    }
    // the compiler must not keep the derived offsets across iterations
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(rows), "+v"(tr0), "+v"(tr1)); }
    __device__ __forceinline__ bf16x8_t row_frag(const char* tile, int ks) const { return *reinterpret_cast<const bf16x8_t*>(tile + (rows ^ (uint32_t)(ks * 32))); }
    __device__ __forceinline__ bf16x8_t tr_frag(const char* tile, int d) const {
        const bf16x4_t lo = seq_tr16(tile + (tr0 ^ (uint32_t)(d * 64))), hi = seq_tr16(tile + (tr1 ^ (uint32_t)(d * 64)));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// A pair of tiles of 64 MUL rows (K and V, or Q and dO) straight into LDS (buffer_load ... lds, 16 B per lane, no registers): a wave fills 1-KiB slabs of consecutive
// LDS, lane l's slot of row l / SW gets the chunk that the swizzle (its own inverse) puts there; slots of chunks behind the head's width get zeros.
// load() asks for the next pair while one is worked on; land() ends the trip in front of the barrier that publishes it.
// KEEP: the lane offsets stay in registers (head widths up to 64: a few); else they are formed anew each time.
template <int DH, int NW, int MUL, bool KEEP>
struct PackedDma {
    using G = PackedGeo<DH>;
    static constexpr int SLABS = MUL * G::TILE / 1024 / NW, ROWS = 1024 / G::PITCH;
    static_assert(MUL * G::TILE / 1024 % NW == 0, "every wave fills the same number of slabs");
    int row0, slot, dim;
    uint32_t pa, pb;                                                            // row strides in bytes
    uint32_t va[KEEP ? SLABS : 1], vb[KEEP ? SLABS : 1];
    __device__ __forceinline__ uint32_t offset(int i, uint32_t pitch) const {
        const int row = row0 + i * ROWS, c = attn_swz<G::SW>(row, slot);
        return c * 8 < dim ? row * pitch + c * 16 : SEQ_OOB;
    }
    __device__ __forceinline__ void init(int wave, int lane, int width, int64_t stride_a, int64_t stride_b) {
        row0 = wave * SLABS * ROWS + lane / G::SW; slot = lane % G::SW; dim = width;
        pa = (uint32_t)(stride_a * 2); pb = (uint32_t)(stride_b * 2);
        if (KEEP)
#pragma unroll
            for (int i = 0; i < SLABS; ++i) { va[i] = offset(i, pa); vb[i] = offset(i, pb); }
    }
    __device__ __forceinline__ void load(int wave, const bf16_t* a, int left_a, char* ta, const bf16_t* b, int left_b, char* tb) {
        if (!KEEP) asm volatile("" : "+v"(row0), "+v"(slot));
#pragma unroll
        for (int i = 0; i < SLABS; ++i) {
            seq_dma16(a, left_a, ta + (wave * SLABS + i) * 1024, KEEP ? va[KEEP ? i : 0] : offset(i, pa));
            seq_dma16(b, left_b, tb + (wave * SLABS + i) * 1024, KEEP ? vb[KEEP ? i : 0] : offset(i, pb));
        }
    }
    __device__ __forceinline__ void land() const { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }      // this wave's slabs; the barrier does the rest
};

// (slot, head) of a block.  Heads fastest, key heads before the query heads that share them: consecutive blocks go round-robin over the 8 XCDs, so with 8, 4, 2 or 1
// key heads an XCD's L2 sees one key head only.
struct PackedBlock { int slot, head, kvh; };
__device__ __forceinline__ PackedBlock packed_block(const PackedArgs& a, int nh) {
    PackedBlock b;
    const int id = (int)blockIdx.x, hi = id % nh;
    b.slot = id / nh;
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

template <typename K>
static inline int packed_launch(K kernel, const PackedArgs& a, int64_t blocks, int threads, int lds, void* stream) {
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

// Few rows: P and dS go into their products with what their rounding left over, too (variants with REST).  Over many rows that rounding makes the error sqrt(2) times that of
// rounding the result alone; over a handful of values it can be any value's worst.  Measured with / without: sequences of 2, 2 and 2 tokens dQ 0.0018 / 0.0026 off in
// norm (the best bf16 result: 0.0018); three snippets of 33 tokens together 5.3 / 5.2 us; a batch of 5720 tokens would pay (forward 43 / 31, dQ 48 / 34, dK and dV 62 / 42 us).
static inline bool packed_exact(const PackedArgs& a) { return a.rows_q <= 256 && a.rows_k <= 256; }

// few enough blocks of 128 rows that blocks half as tall (head widths up to 64), whose chain of steps takes half as long, pay: see the rules where it is called
static inline bool packed_few(int rows, int heads, int64_t most) { return (int64_t)(rows / 128) * heads <= most; }

int packed_dkv_run(PackedArgs& a, void* stream);     // packed_attention_dkv.hip
