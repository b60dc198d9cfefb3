// Backward of packed causal attention, dK and dV (see packed_attention.hip for the formulas and the walk).
//
// A wave owns 32 KT keys of one key head and walks the query rows that see them, head after head of the group -- the sum over the group's heads happens in
// the accumulators, in a fixed order.  S = Q K^T (lane = key): P and dS are operand-shaped for dV^T = dO^T P and dK^T = Q^T dS.  The rows' -lse / scale and
// -delta are the accumulators' INPUT, read from LDS beside the tile, so that P = exp2(c S) and dS = P dP cost one multiplication each.
//
// Head widths above 64: KT = 2 and ONE wave per SIMD.  dK and dV take 256 accumulator registers (the AGPR half of the file), the K fragments, S, dP, P and dS 160 of the
// others; the V fragments, which would be 64 more, wait in LDS (129 of 160 KB: one block per CU anyway).  Every Q / dO fragment read from LDS feeds two
// products, and with 64 products per 32 rows the matrix pipe has work while the exponentials run.  At 32 keys per wave and two waves per SIMD, K, V, dK and
// dV take 192 of 256 registers, which leaves one fragment in flight, and every product waits out an LDS read.
// Head widths up to 64: KT = 1, three waves per SIMD hide each other's latencies.
#include "packed_common.h"

template <int DH, int KT, int RG, int WPE, bool VLDS, bool REST>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) packed_dkv_kernel(const PackedArgs a) {
    using G = PackedGeo<DH>;
    constexpr int NW = 4, KG = NW / RG, BN = 32 * KT * KG, NT = 64 * NW, STAGE = 2 * G::TILE + 512;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int kvh = (int)blockIdx.x % a.hkv, part = (int)blockIdx.x / a.hkv % a.nsplit, slot = (int)blockIdx.x / a.hkv / a.nsplit, group = a.hq / a.hkv;
    const SeqSlot s = seq_find_longest<BN, true>(a.cu_k, a.nseq, a.rows_k, slot, a.nslots);
    if (s.tile < 0 || s.tile * BN >= s.len) return;
    if (s.seq == a.nseq) {
        if (a.nsplit > 1) return;                                               // (the reduction writes those rows)
        packed_zero_rows<BN, NT>(a.dk, a.hkv, a.dim, s, kvh);
        packed_zero_rows<BN, NT>(a.dv, a.hkv, a.dim, s, kvh);
        return;
    }
    const int qstart = seq_cu(a.cu_q, s.seq, a.rows_q), qlen = max(0, seq_cu(a.cu_q, s.seq + 1, a.rows_q) - qstart);
    const int shift = s.len - qlen;                                             // key j is seen by rows i >= j - shift
    const int kg = wave % KG, rg = wave / KG;                                   // this wave's keys and, RG = 2, its half of each tile's rows
    const int j0 = s.tile * BN + kg * 32 * KT, kj = j0 + (lane & 31);
    const int first = max(0, s.tile * BN - shift) & ~63;                        // first query row the block needs, on a tile border
    const int w_first = j0 - shift;
    const int tiles = max(0, (qlen - first + 63) >> 6);
    const int64_t all = (int64_t)tiles * group;                                 // (head, tile) steps; this block takes its part of them
    const int i0 = (int)(all * part / a.nsplit), i1 = (int)(all * (part + 1) / a.nsplit);

    PackedLane<DH> at;
    at.init(lane);
    char* vt_ = smem + 2 * STAGE + wave * KT * 32 * G::PITCH;                   // VLDS: this wave's V rows, laid out like a staged tile
    bf16x8_t kf[KT][G::KS], vf[VLDS ? 1 : KT][G::KS];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int64_t krow = s.start + kj + 32 * kt;
        packed_row_frags<DH>(kf[kt], a.k + krow * a.k_row + kvh * a.k_head, kj + 32 * kt < s.len, a.dim);
        packed_row_frags<DH>(vf[VLDS ? 0 : kt], a.v + krow * a.v_row + kvh * a.v_head, kj + 32 * kt < s.len, a.dim);
        if (VLDS)
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) *reinterpret_cast<bf16x8_t*>(vt_ + kt * 32 * G::PITCH + (at.rows ^ (uint32_t)(ks * 32))) = vf[0][ks];
    }
    f32x16_t dk[KT][G::DT], dv[KT][G::DT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int d = 0; d < G::DT; ++d) dk[kt][d] = dv[kt][d] = packed_splat(0.f);
    // (scales under 1e-36 count as 1e-36 in the exponent, where neither leaves anything of a score: lse / scale stays an fp32 number)
    const float es = fmaxf(a.scale, 1e-36f), c2 = es * 1.4426950408889634f, inv_scale = 1.f / es;

    PackedDma<DH, NW, 1, false> st;
    st.init(wave, lane, a.dim, a.q_row, a.g_row);
    float stat = 0.f;                                                           // threads 0..63: -lse / scale, 64..127: -delta of the tile's rows
    auto load = [&](int i) {
        const int head = kvh * group + i / tiles, r0 = first + (i % tiles) * 64;
        const bf16_t* qp = a.q + (int64_t)(qstart + r0) * a.q_row + head * a.q_head;
        const bf16_t* gp = a.dout + (int64_t)(qstart + r0) * a.g_row + head * a.g_head;
        char* to = smem + (i & 1) * STAGE;
        st.load(wave, qp, seq_bytes_left(qlen - r0, a.q_row * 2, a.dim), to, gp, seq_bytes_left(qlen - r0, a.g_row * 2, a.dim), to + G::TILE);
        if (tid < 128) {
            const int row = r0 + (tid & 63);
            const int64_t at = (int64_t)head * a.rows_q + qstart + row;
            stat = tid < 64 ? -INFINITY : 0.f;
            if (row < qlen) {
                const float x = tid < 64 ? a.lse[at] : a.delta[at];
                stat = tid >= 64 ? -x : (x == -INFINITY ? -INFINITY : -x * inv_scale);
            }
        }
    };

    // 32 query rows rbase .. of the staged tile
    auto rows32 = [&](const char* qt_, const char* gt_, const float* stats, int rbase) {
        f32x16_t sacc[KT], dp[KT];                                              // start at -lse / scale and -delta: p = exp2(c2 S), dS = p dP
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(stats + 8 * g + 4 * h), y = *reinterpret_cast<const f32x4_t*>(stats + 64 + 8 * g + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) { sacc[kt][4 * g + e] = x[e]; dp[kt][4 * g + e] = y[e]; }
        }
        if constexpr (VLDS) {
            // Four runs of products -- S, dP with the exponentials, dV with dS, dK -- as one chain of stages of KT products.  A stage's LDS fragments are requested in the stage
            // before, and the compiler may not move them back behind its products: with one wave per SIMD nobody else hides their latency (4 x 4096 rows, 16 / 4 heads:
            // 600 us; in the order below 700; requested two stages ahead 605).
            static_assert(!REST, "weights are one bf16 value here");
            constexpr int KS = G::KS, DT = G::DT, NS = 2 * KS + 4 * DT, N = 16 * KT;
            bf16x8_t fr[NS], vr[KT][KS], pf[KT][2], ds[KT][2];
            auto fetch = [&](int n) __attribute__((always_inline)) {
                if (n < KS) fr[n] = at.row_frag(qt_, n);
                else if (n < 2 * KS) {
                    fr[n] = at.row_frag(gt_, n - KS);
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) vr[kt][n - KS] = at.row_frag(vt_ + kt * 32 * G::PITCH, n - KS);
                } else if (n < 2 * KS + 2 * DT) fr[n] = at.tr_frag(gt_ + (n - 2 * KS) / DT * 16 * G::PITCH, (n - 2 * KS) % DT);
                else if (n < NS) fr[n] = at.tr_frag(qt_ + (n - 2 * KS - 2 * DT) / DT * 16 * G::PITCH, (n - 2 * KS) % DT);
            };
            fetch(0);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                fetch(n + 1);
                __builtin_amdgcn_sched_barrier(0);
                if (n < KS) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) sacc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n], kf[kt][n], sacc[kt], 0, 0, 0);
                    if (n == KS - 1 && rbase < w_first + 32 * KT - 1) {             // some of these rows do not see all of the wave's keys
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            int lim = kj + 32 * kt - shift - rbase - 4 * h;         // rows below do not see this lane's key
                            asm volatile("" : "+v"(lim));
#pragma unroll
                            for (int r = 0; r < 16; ++r) sacc[kt][r] = seq_crow(r) >= lim ? sacc[kt][r] : -INFINITY;
                        }
                    }
                } else if (n < 2 * KS) {
                    const int ks = n - KS;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) dp[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n], vr[kt][ks], dp[kt], 0, 0, 0);
#pragma unroll
                    for (int e = ks * N / KS; e < (ks + 1) * N / KS; ++e) {
                        sacc[e / 16][e % 16] = __builtin_amdgcn_exp2f(sacc[e / 16][e % 16] * c2);
                        if (e % 8 == 7) {
                            const int kt = e / 16, s2 = e / 8 % 2;
                            const float p[8] = {sacc[kt][8 * s2], sacc[kt][8 * s2 + 1], sacc[kt][8 * s2 + 2], sacc[kt][8 * s2 + 3], sacc[kt][8 * s2 + 4], sacc[kt][8 * s2 + 5],
                                                sacc[kt][8 * s2 + 6], sacc[kt][8 * s2 + 7]};
                            pf[kt][s2] = seq_pack8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
                        }
                    }
                } else if (n < 2 * KS + 2 * DT) {
                    const int i = n - 2 * KS, s2 = i / DT, d = i % DT;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) dv[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n], pf[kt][s2], dv[kt][d], 0, 0, 0);
#pragma unroll
                    for (int e = i * N / (2 * DT); e < (i + 1) * N / (2 * DT); ++e) {
                        dp[e / 16][e % 16] *= sacc[e / 16][e % 16];
                        if (e % 8 == 7) {
                            const int kt = e / 16, s2 = e / 8 % 2;
                            const float x[8] = {dp[kt][8 * s2], dp[kt][8 * s2 + 1], dp[kt][8 * s2 + 2], dp[kt][8 * s2 + 3], dp[kt][8 * s2 + 4], dp[kt][8 * s2 + 5],
                                                dp[kt][8 * s2 + 6], dp[kt][8 * s2 + 7]};
                            ds[kt][s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
                        }
                    }
                } else {
                    const int i = n - 2 * KS - 2 * DT, s2 = i / DT, d = i % DT;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) dk[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n], ds[kt][s2], dk[kt][d], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                const bf16x8_t qa = at.row_frag(qt_, ks), ga = at.row_frag(gt_, ks);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    sacc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qa, kf[kt][ks], sacc[kt], 0, 0, 0);
                    dp[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ga, vf[kt][ks], dp[kt], 0, 0, 0);
                }
            }
            if (rbase < w_first + 32 * KT - 1) {                                    // some of these rows do not see all of the wave's keys
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    int lim = kj + 32 * kt - shift - rbase - 4 * h;                 // rows below do not see this lane's key
                    asm volatile("" : "+v"(lim));
#pragma unroll
                    for (int r = 0; r < 16; ++r) sacc[kt][r] = seq_crow(r) >= lim ? sacc[kt][r] : -INFINITY;
                }
            }
            bf16x8_t pf[KT][2], ds[KT][2], pr[REST ? KT : 1][2], dr[REST ? KT : 1][2];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    float p[8], x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int r = 8 * s2 + e;
                        p[e] = __builtin_amdgcn_exp2f(sacc[kt][r] * c2);
                        x[e] = p[e] * dp[kt][r];
                    }
                    pf[kt][s2] = seq_pack8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
                    ds[kt][s2] = seq_pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
                    if (REST) {
                        pr[REST ? kt : 0][s2] = seq_rest8(p, pf[kt][s2]);
                        dr[REST ? kt : 0][s2] = seq_rest8(x, ds[kt][s2]);
                    }
                }
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int d = 0; d < G::DT; ++d) {
                    const bf16x8_t gt = at.tr_frag(gt_ + s2 * 16 * G::PITCH, d), qt = at.tr_frag(qt_ + s2 * 16 * G::PITCH, d);
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        if (REST) {
                            dv[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gt, pr[REST ? kt : 0][s2], dv[kt][d], 0, 0, 0);
                            dk[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt, dr[REST ? kt : 0][s2], dk[kt][d], 0, 0, 0);
                        }
                        dv[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gt, pf[kt][s2], dv[kt][d], 0, 0, 0);
                        dk[kt][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt, ds[kt][s2], dk[kt][d], 0, 0, 0);
                    }
                }
        }
    };

    if (i0 < i1) load(i0);
    for (int i = i0; i < i1; ++i) {
        char* qt_ = smem + (i & 1) * STAGE;
        char* gt_ = qt_ + G::TILE;
        float* stats = reinterpret_cast<float*>(gt_ + G::TILE);
        if (tid < 128) stats[tid] = stat;
        st.land();
        __syncthreads();
        if (i + 1 < i1) load(i + 1);
        const int r0 = first + (i % tiles) * 64;
        if (r0 + (RG == 2 ? rg * 32 + 31 : 63) < w_first) continue;             // (wave-uniform) none of these rows sees this wave's keys
        at.forget();
#pragma unroll 1
        for (int qt = RG == 2 ? rg : 0; qt < (RG == 2 ? rg + 1 : 2); ++qt) rows32(qt_ + qt * 32 * G::PITCH, gt_ + qt * 32 * G::PITCH, stats + qt * 32, r0 + qt * 32);
    }
    if constexpr (RG == 2) {                                                    // the row halves' sums meet in LDS, register by register
        static_assert(KT == 1, "one set of accumulators");
        __syncthreads();
        float* xs = reinterpret_cast<float*>(smem) + kg * 2 * G::DT * 16 * 64 + lane;
        if (rg == 1)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    xs[(d * 32 + e) * 64] = dk[0][d][e];
                    xs[(d * 32 + 16 + e) * 64] = dv[0][d][e];
                }
        __syncthreads();
        if (rg == 0)
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    dk[0][d][e] += xs[(d * 32 + e) * 64];
                    dv[0][d][e] += xs[(d * 32 + 16 + e) * 64];
                }
    }
    if (a.nsplit > 1) {                                                         // fp32 parts, 16 B per lane and store
        if (rg != 0) return;
        float* pk = a.part + (((int64_t)part * 2 * a.rows_k + s.start) * a.hkv + kvh) * a.dim;
        float* pv = pk + (int64_t)a.rows_k * a.hkv * a.dim;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const int j = kj + 32 * kt;
            if (j >= s.len) continue;
            const int64_t at = (int64_t)j * a.hkv * a.dim;
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int col = 32 * d + 8 * g + 4 * h;
                    if (col < a.dim) {
                        *reinterpret_cast<f32x4_t*>(pk + at + col) = f32x4_t{dk[kt][d][4 * g], dk[kt][d][4 * g + 1], dk[kt][d][4 * g + 2], dk[kt][d][4 * g + 3]};
                        *reinterpret_cast<f32x4_t*>(pv + at + col) = f32x4_t{dv[kt][d][4 * g], dv[kt][d][4 * g + 1], dv[kt][d][4 * g + 2], dv[kt][d][4 * g + 3]};
                    }
                }
        }
        return;
    }
    __syncthreads();
    if (rg != 0) return;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int j = j0 + 32 * kt;
        if (j >= s.len) break;
        const int64_t to = ((int64_t)(s.start + j) * a.hkv + kvh) * a.dim;
        char* region = smem + wave * 32 * G::PITCH;                             // (one region per wave: LDS serves a wave's accesses in order)
        packed_write_rows<DH>(region, dk[kt], a.scale, a.dk + to, (int64_t)a.hkv * a.dim, min(32, s.len - j), a.dim);
        packed_write_rows<DH>(region, dv[kt], 1.f, a.dv + to, (int64_t)a.hkv * a.dim, min(32, s.len - j), a.dim);
    }
}

// dK, dV <- the parts' sums in order, rounded once; zeros behind the last sequence
__global__ void __launch_bounds__(256) packed_dkv_sum_kernel(const PackedArgs a) {
    const int64_t n = (int64_t)a.rows_k * a.hkv * a.dim, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) return;
    const bool live = i / (a.hkv * a.dim) < seq_cu(a.cu_k, a.nseq, a.rows_k);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live)
            for (int p = 0; p < a.nsplit; ++p) {
                const float* src = a.part + (int64_t)(2 * p + m) * n + i;
                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(src), y = *reinterpret_cast<const f32x4_t*>(src + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { f[e] += x[e]; f[4 + e] += y[e]; }
            }
        if (m == 0)
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= a.scale;
        *reinterpret_cast<u32x4_t*>((m ? a.dv : a.dk) + i) = pack8(f);
    }
}

// Parts that a key tile's (head, row tile) steps are cut into.  A launch takes the longest chain of steps (all sequences taken as equally long), or the time that all pairs take on a
// full chip, whichever is longer; parts shorten the chain and cost a second launch and their fp32 sums written and read.  The rates are
// measured: a step 1 us (64 keys per block), 2 us (128) or 4.2 us (256, width 128), 0.56 or 1 us per million pairs, 5 us, 6 TB/s.  The model agreed with the measured order
// of n = 1 .. 8 on ten batches, e.g. 4 x 700 rows, 8 / 8 heads of width 64, n = 1, 2, 3: 33 / 40 / 44 us the whole backward; 16 / 4 heads, n = 3, 4, 5, 8: 57 / 55 / 56 / 64.
static int packed_dkv_splits(int nseq, int rows_q, int rows_k, int hq, int hkv, int dim) {
    if (rows_q == 0 || rows_k == 0) return 1;                                   // zeros: nothing to cut
    const float length = (float)rows_q / (float)(nseq > 0 ? nseq : 1);
    const float step = dim > 64 ? 4.2f * (float)dim / 128.f : packed_few(rows_q, hq, 512) ? 1.f : 2.f;
    const float chain = (length / 64.f + 1.f) * (float)(hq / hkv) * step;
    const float all = (float)rows_q * length * 0.5f * (float)hq * (dim > 64 ? 1e-6f : 0.56e-6f);
    const float part = (float)rows_k * (float)hkv * (float)dim * 16.f / 6e6f;
    int best = 1;
    float least = 0.f;
    for (int n = 1; n <= 8; ++n) {
        const float t = (chain / (float)n > all ? chain / (float)n : all) + (n > 1 ? 5.f + (float)n * part : 0.f);
        if (n == 1 || t < least) {
            least = t;
            best = n;
        }
    }
    return best;
}
extern "C" int64_t genie_packed_attention_bwd_ws_floats(int nseq, int rows_q, int rows_k, int hq, int hkv, int dim) {
    if (nseq < 0 || rows_q < 0 || rows_k < 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || dim <= 0) return 0;
    const int n = packed_dkv_splits(nseq, rows_q, rows_k, hq, hkv, dim);
    return (int64_t)hq * rows_q + 4 + (n > 1 ? (int64_t)2 * n * rows_k * hkv * dim : 0);      // delta (rounded up to 16 B; written without keys, too), parts
}

template <int DH, int KT, int RG, int WPE, bool REST = false>
static int packed_dkv_dispatch(PackedArgs& a, void* stream) {
    constexpr bool VLDS = KT > 1;
    a.nslots = a.rows_k / (128 * KT / RG) + a.nseq + 1;
    const int rc = packed_launch(packed_dkv_kernel<DH, KT, RG, WPE, VLDS, REST>, a, (int64_t)a.nslots * a.hkv * a.nsplit, 256,
                                 4 * PackedGeo<DH>::TILE + 1024 + (VLDS ? 128 * KT * PackedGeo<DH>::PITCH : 0), stream);
    if (rc != GENIE_OK || a.nsplit == 1) return rc;
    return packed_launch(packed_dkv_sum_kernel, a, ((int64_t)a.rows_k * a.hkv * a.dim / 8 + 255) / 256, 256, 0, stream);
}
int packed_dkv_run(PackedArgs& a, void* stream) {
    a.nsplit = packed_dkv_splits(a.nseq, a.rows_q, a.rows_k, a.hq, a.hkv, a.dim);
    a.part = a.delta + ((int64_t)a.hq * a.rows_q + 3) / 4 * 4;
    if (packed_exact(a)) {
        if (a.dim <= 32) return packed_dkv_dispatch<32, 1, 2, 1, true>(a, stream);
        if (a.dim <= 64) return packed_dkv_dispatch<64, 1, 2, 1, true>(a, stream);
        if (a.dim <= 96) return packed_dkv_dispatch<96, 1, 1, 1, true>(a, stream);
        return packed_dkv_dispatch<128, 1, 1, 1, true>(a, stream);
    }
    if (packed_few(a.rows_q, a.hq, 512)) {
        if (a.dim <= 32) return packed_dkv_dispatch<32, 1, 2, 3>(a, stream);
        if (a.dim <= 64) return packed_dkv_dispatch<64, 1, 2, 3>(a, stream);
    }
    if (a.dim <= 32) return packed_dkv_dispatch<32, 1, 1, 3>(a, stream);
    if (a.dim <= 64) return packed_dkv_dispatch<64, 1, 1, 3>(a, stream);
    if (a.dim <= 96) return packed_dkv_dispatch<96, 2, 1, 1>(a, stream);
    return packed_dkv_dispatch<128, 2, 1, 1>(a, stream);
}
