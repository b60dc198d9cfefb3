// Softmax attention of ONE new token per sequence against its key / value cache (grouped heads), optionally appending the token's key and value.
//
//   o = softmax(scale q . K[0..n]) V[0..n],   n = lengths[b] (the new token's own place) or n = lengths[b] - 1 without a new token
//
// Bound by reading K and V once: 4 n Hkv D bytes against 4 n Hq D operations.  The query heads that share a key head are the 16 columns of one
// 16x16x32 product, so a cache row is read once for all of them and the vector units do no dot products; a wave walks 32-key tiles on its own --
// loaded as whole rows, K and then V through its private LDS tile into operand layout, the next tile's loads in flight from the first product on -- and there is
// no barrier in the key loop.  (64 sequences of up to 8191 keys, 4 key heads of width 128, 512 MB, cold: 93 us = 5.5 TB/s,
// parts joined in another 5.  Call 97 us, without the non-temporal hint 108; with K straight into operand registers, 64 B of each of 16 rows per load, the kernel took 104 for 88.)  Where batch x key heads do not fill the chip, short caches get blocks of more waves (their parts meet in LDS), long ones are
// split over blocks, and a second small kernel joins the parts (maximum, sum, unnormalised fp32 output) in a fixed order.  Lengths are read on the device: a captured graph replays with the lengths of the day.
#include "seq_common.h"
#include "genie_hip.h"

struct CachedArgs {
    const bf16_t *q, *k_new, *v_new;
    bf16_t *kc, *vc, *out;
    const int32_t* lengths;
    float *part_ml, *part_o;       // [B][Hq][nsplit][2], [B][Hq][nsplit][dim]
    int batch, hq, hkv, dim, cap, nsplit, hgroups;
    int64_t q_b, q_h, kn_b, kn_h, vn_b, vn_h, k_b, k_t, k_h, v_b, v_t, v_h;
    float scale;
};

template <int DH>
constexpr int cached_wave_bytes() {                                             // one wave's V tile, later its output part, rows padded by 16 B against bank conflicts
    const int tile = 32 * (DH <= 64 ? 128 : 256), part = 16 * (DH + 4) * 4;
    return tile > part ? tile : part;
}

template <int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? 4 : 2) cached_step_kernel(const CachedArgs a) {
    constexpr int KS = DH / 32, DT = DH / 16, CPR = DH / 8, PITCH = DH <= 64 ? 128 : 256, SW = PITCH / 16, VP = 32 * CPR / 64;
    constexpr int WREG = cached_wave_bytes<DH>();
    extern __shared__ __attribute__((aligned(16))) char smem[];                 // NW WREG + 128 NW
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    int id = (int)blockIdx.x;
    const int kvh = id % a.hkv; id /= a.hkv;
    const int hg = id % a.hgroups; id /= a.hgroups;
    const int split = id % a.nsplit, b = id / a.nsplit;
    const int group = a.hq / a.hkv;
    const int hsub = hg * 16 + col;                                             // this lane's query head inside the group
    const bool has_head = hsub < group;
    const int head = kvh * group + (has_head ? hsub : 0);
    const int given = a.lengths[b];
    const bool append = a.k_new != nullptr;
    const bool bad = given > a.cap - (append ? 1 : 0);                          // no room: the row says so with NaN
    const bool idle = given < 0 || (given == 0 && !append);                     // an unused row of the batch: zeros
    const int n = bad || idle ? 0 : given;

    bf16x8_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0};
        const int d = ks * 32 + g * 8;
        if (has_head && d < a.dim) qf[ks] = *reinterpret_cast<const bf16x8_t*>(a.q + b * a.q_b + head * a.q_h + d);
    }
    const float c2 = a.scale * 1.4426950408889634f;
    char* vt = smem + wave * WREG;
    // a tile's rows in 16-B pieces, 64 / CPR rows per load; K and V have their own row strides.  Where whole rows fill a load (EVEN) a lane's pieces lie in one column a
    // constant number of rows apart, and one register of each kind is enough: the swizzle's key of row r + R i is that of r with the key of R i flipped in.
    constexpr bool EVEN = 64 % CPR == 0;
    constexpr int R = 64 / CPR, NO = EVEN ? 1 : VP;
    uint32_t koff[NO], voff[NO], lds[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) {
        const int idx = i * 64 + lane, row = idx / CPR, c = idx % CPR;
        koff[i] = c * 8 < a.dim ? (uint32_t)(row * a.k_t * 2) + c * 16 : SEQ_OOB;
        voff[i] = c * 8 < a.dim ? (uint32_t)(row * a.v_t * 2) + c * 16 : SEQ_OOB;
        lds[i] = (uint32_t)(row * PITCH + (attn_swz<SW>(row, c) << 4));
    }
    auto lds_at = [&](int i) { return EVEN ? (lds[0] ^ (uint32_t)(attn_swz<SW>(i * R, 0) << 4)) + i * R * PITCH : lds[EVEN ? 0 : i]; };
    auto koff_at = [&](int i) { return EVEN ? koff[0] + (uint32_t)(i * R * (int)a.k_t * 2) : koff[EVEN ? 0 : i]; };      // (SEQ_OOB plus a tile stays out of range)
    auto voff_at = [&](int i) { return EVEN ? voff[0] + (uint32_t)(i * R * (int)a.v_t * 2) : voff[EVEN ? 0 : i]; };
    const uint32_t roff = (uint32_t)(col * PITCH + (attn_swz<SW>(col, g) << 4));   // operand fragment of a row: chunk 4 ks + g is this with bits 6.. flipped
    uint32_t toff[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int row = 4 * g + ((lane >> 2) & 3), c = d * 16 + 4 * (lane & 3);
        toff[d] = (uint32_t)(row * PITCH + (attn_swz<SW>(row, c >> 3) << 4) + (c & 7) * 2);
    }

    f32x4_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, mc = 0.f, l_run = 0.f;

    u32x4_t kr[VP], vr[VP];
    // scores of the up to 32 keys in kr (`live` of them exist); V to LDS behind them: kr and vr are free then.  (LDS serves a wave's accesses in order: K's
    // fragments are read before V overwrites them.)
    auto scores = [&](f32x4_t (&s)[2], int live) {
#pragma unroll
        for (int i = 0; i < VP; ++i) *reinterpret_cast<u32x4_t*>(vt + lds_at(i)) = kr[i];
        bf16x8_t kf[2][KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) kf[kt][ks] = *reinterpret_cast<const bf16x8_t*>(vt + kt * 16 * PITCH + (roff ^ (uint32_t)(ks * 64)));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < VP; ++i) *reinterpret_cast<u32x4_t*>(vt + lds_at(i)) = vr[i];
        s[0] = s[1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt][ks], qf[ks], s[kt], 0, 0, 0);
        if (live < 32) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[kt][e] = kt * 16 + 4 * g + e < live ? s[kt][e] : -INFINITY;
        }
    };
    auto weigh = [&](const f32x4_t (&s)[2]) {
        float p[8], ps;
        bool with_max = m_run == -INFINITY;                                     // (the same in the four lanes of a column; decided for the wave below)
        for (;;) {
            if (__builtin_amdgcn_ballot_w64(with_max) != 0) {
                float tm = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
                tm = fmaxf(tm, __shfl_xor(tm, 16));
                tm = fmaxf(tm, __shfl_xor(tm, 32));
                const float m_new = fmaxf(m_run, tm), mc_new = m_new == -INFINITY ? 0.f : m_new * c2;
                const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - mc_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][e] *= alpha;
                m_run = m_new;
                mc = mc_new;
            }
            ps = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], c2, -mc));
                ps += p[e];
            }
            if (__builtin_amdgcn_ballot_w64(with_max) != 0 || __builtin_amdgcn_ballot_w64(!(ps <= 256.f)) == 0) break;
            with_max = true;
        }
        l_run += ps;
        // P and what its rounding left over: the second product hides behind the loads, and no rounding but the output's is left
        const bf16x8_t pf = seq_pack8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]), pr = seq_rest8(p, pf);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const bf16x4_t lo = seq_tr16(vt + toff[d]), hi = seq_tr16(vt + toff[d] + 16 * PITCH);
            const bf16x8_t vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pr, acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, acc[d], 0, 0, 0);
        }
    };

    const int tiles = (n + 31) >> 5, per = (tiles + a.nsplit - 1) / a.nsplit, t_end = min(tiles, (split + 1) * per);
    const bf16_t* kb = a.kc + b * a.k_b + kvh * a.k_h;
    const bf16_t* vb = a.vc + b * a.v_b + kvh * a.v_h;
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < NO; ++i) asm volatile("" : "+v"(koff[i]), "+v"(voff[i]), "+v"(lds[i]));      // (derived offsets are formed anew)
        const bf16_t* kp = kb + (int64_t)t * 32 * a.k_t;
        const bf16_t* vp = vb + (int64_t)t * 32 * a.v_t;
        const int kl = seq_bytes_left(n - t * 32, a.k_t * 2, a.dim), vl = seq_bytes_left(n - t * 32, a.v_t * 2, a.dim);
#pragma unroll
        for (int i = 0; i < VP; ++i) kr[i] = seq_load16<true>(kp, kl, koff_at(i));
#pragma unroll
        for (int i = 0; i < VP; ++i) vr[i] = seq_load16<true>(vp, vl, voff_at(i));
    };
    if (append && split == 0 && wave == NW - 1 && !bad && !idle) {
        // the new token, in the wave with the fewest tiles: a tile of one key, taken from the arguments and put into the cache by the same lanes (no other lane of this launch reads that row)
        const bf16_t* kp = a.k_new + b * a.kn_b + kvh * a.kn_h;
        const bf16_t* vp = a.v_new + b * a.vn_b + kvh * a.vn_h;
        bf16_t* kd = a.kc + b * a.k_b + kvh * a.k_h + (int64_t)n * a.k_t;
        bf16_t* vd = a.vc + b * a.v_b + kvh * a.v_h + (int64_t)n * a.v_t;
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int idx = i * 64 + lane, row = idx / CPR, c = idx % CPR;
            kr[i] = vr[i] = u32x4_t{0, 0, 0, 0};
            if (row == 0 && c * 8 < a.dim) {
                kr[i] = *reinterpret_cast<const u32x4_t*>(kp + c * 8);
                vr[i] = *reinterpret_cast<const u32x4_t*>(vp + c * 8);
                if (hg == 0) {
                    *reinterpret_cast<u32x4_t*>(kd + c * 8) = kr[i];
                    *reinterpret_cast<u32x4_t*>(vd + c * 8) = vr[i];
                }
            }
        }
        f32x4_t s[2];
        scores(s, 1);
        weigh(s);
    }
    int t = split * per + wave;
    if (t < t_end) load(t);
    while (t < t_end) {
        f32x4_t s[2];
        scores(s, min(32, n - t * 32));
        t += NW;
        if (t < t_end) load(t);                                                 // in flight under the exponentials and the second product
        weigh(s);
    }
    // the waves' parts: maxima, sums, outputs through LDS
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    float* ml = reinterpret_cast<float*>(smem + NW * WREG);
    float* ob = reinterpret_cast<float*>(smem + wave * WREG);                   // this wave's own tile region: [16 heads][DH + 4]
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_t*>(ob + col * (DH + 4) + d * 16 + 4 * g) = acc[d];
    if (g == 0) {
        ml[(wave * 16 + col) * 2] = m_run == -INFINITY ? -INFINITY : mc;
        ml[(wave * 16 + col) * 2 + 1] = l_run;
    }
    __syncthreads();
    const int nh = min(16, group - hg * 16), vec = a.dim / 4;
    for (int i = tid; i < nh * vec; i += 64 * NW) {
        const int hh = i / vec, d = (i % vec) * 4, ho = kvh * group + hg * 16 + hh;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[(w * 16 + hh) * 2]);
        float l = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = ml[(w * 16 + hh) * 2], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
            const float lw = ml[(w * 16 + hh) * 2 + 1];
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(smem + w * WREG) + hh * (DH + 4) + d);
            if (mw != -INFINITY || lw != 0.f) {                                 // (a wave that saw only NaN keeps its NaN)
                l += lw * (mw == -INFINITY ? 1.f : f);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += x[e] * (mw == -INFINITY ? 1.f : f);
            }
        }
        if (a.nsplit == 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            u32x2_t w = {pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
            if (bad) w = u32x2_t{0x7fc07fc0u, 0x7fc07fc0u};
            *reinterpret_cast<u32x2_t*>(a.out + ((int64_t)b * a.hq + ho) * a.dim + d) = w;
        } else {
            const int64_t at = ((int64_t)b * a.hq + ho) * a.nsplit + split;
            *reinterpret_cast<f32x4_t*>(a.part_o + at * a.dim + d) = o;
            if (d == 0) {
                a.part_ml[at * 2] = m;
                a.part_ml[at * 2 + 1] = bad ? __builtin_nanf("") : l;
            }
        }
    }
}

// Join of the parts of one (sequence, head): a thread per 4 columns and part group; the group sums are added in a fixed order.
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedArgs a) {
    __shared__ float sm[256 * 4 + 8], sl[256], smax[4];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x;
    const float* ml = a.part_ml + bh * a.nsplit * 2;
    const float* po = a.part_o + bh * a.nsplit * a.dim;
    float m = -INFINITY;
    for (int s = tid; s < a.nsplit; s += 256) m = fmaxf(m, ml[2 * s]);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
    if ((tid & 63) == 0) smax[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    const int vec = a.dim / 4, ng = 256 / vec, grp = tid / vec, d = (tid % vec) * 4;
    float l = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    if (grp < ng)
        for (int s = grp; s < a.nsplit; s += ng) {
            const float ms = ml[2 * s], f = ms == -INFINITY ? (ml[2 * s + 1] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(ms - m);
            if (f == 0.f) continue;                                             // an empty part
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(po + (int64_t)s * a.dim + d);
            l += ml[2 * s + 1] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += x[e] * f;
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) sm[tid * 4 + e] = o[e];
    sl[tid] = l;
    __syncthreads();
    if (tid < vec) {
        for (int j = 1; j < ng; ++j) {
            l += sl[j * vec + tid];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += sm[(j * vec + tid) * 4 + e];
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;                             // (NaN stays NaN: a length the cache cannot hold)
        const u32x2_t w = {pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2_t*>(a.out + bh * a.dim + d) = w;
    }
}

// waves of a block that takes a whole short cache, four tiles of 32 keys each
static int cached_wide(int dim) { return dim <= 64 ? 16 : 8; }
// parts of the key axis (0: one part, a wide block)
static int cached_splits(int batch, int hq, int hkv, int dim, int cap) {
    const int64_t base = (int64_t)batch * hkv * ((hq / hkv + 15) / 16);
    if (base < 512 && cap <= 128 * cached_wide(dim)) return 0;
    int64_t n = base > 0 ? (2048 + base - 1) / base : 1;
    const int64_t most = (cap + 127) / 128;
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : n > 128 ? 128 : n);
}

extern "C" int64_t genie_cached_attention_ws_floats(int batch, int hq, int hkv, int dim, int capacity) {
    if (batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || dim <= 0 || capacity <= 0) return 0;
    const int n = cached_splits(batch, hq, hkv, dim, capacity);
    return n <= 1 ? 0 : (int64_t)batch * hq * n * (dim + 4);
}

template <int DH>
static int cached_dispatch(CachedArgs& a, void* stream) {
    constexpr int NWIDE = DH <= 64 ? 16 : 8, WREG = cached_wave_bytes<DH>();
    const bool wide = a.nsplit == 0;
    a.nsplit = wide ? 1 : a.nsplit;
    const int64_t blocks = (int64_t)a.batch * a.hkv * a.hgroups * a.nsplit;
    GENIE_CHECK_ARG(blocks < (1ll << 31), "genie_cached_attention_step: too many blocks");
    const int nw = wide ? NWIDE : 4, lds = nw * (WREG + 128);
    auto* kernel = wide ? cached_step_kernel<DH, NWIDE> : cached_step_kernel<DH, 4>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) {
            genie_set_error("genie_cached_attention_step: %s", hipGetErrorString(e));
            return GENIE_ERR_HIP;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * nw), lds, (hipStream_t)stream, a);
    GENIE_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        hipLaunchKernelGGL(cached_join_kernel, dim3((unsigned)(a.batch * a.hq)), dim3(256), 0, (hipStream_t)stream, a);
        GENIE_CHECK_LAUNCH();
    }
    return GENIE_OK;
}

extern "C" int genie_cached_attention_step(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache, const int32_t* lengths, void* out,
                                           float* ws, int64_t ws_floats, int batch, int hq, int hkv, int dim, int capacity, const int64_t* q_strides,
                                           const int64_t* kn_strides, const int64_t* vn_strides, const int64_t* kc_strides, const int64_t* vc_strides, float scale,
                                           void* stream) {
    const char* what = "genie_cached_attention_step";
    GENIE_CHECK_ARG(q && k_cache && v_cache && lengths && out && q_strides && kc_strides && vc_strides, "%s: null pointer", what);
    GENIE_CHECK_ARG(!k_new == !v_new, "%s: a new key needs a new value", what);
    GENIE_CHECK_ARG(!k_new || (kn_strides && vn_strides), "%s: null strides", what);
    GENIE_CHECK_ARG(batch > 0 && capacity > 0 && hkv > 0 && hq > 0 && hq % hkv == 0, "%s: bad sizes (batch %d, capacity %d, heads %d / %d)", what, batch, capacity, hq, hkv);
    GENIE_CHECK_ARG(dim > 0 && dim % 8 == 0 && dim <= 128, "%s: head width %d (a multiple of 8 up to 128 is supported)", what, dim);
    GENIE_CHECK_ARG(scale > 0.f && scale < 1e30f, "%s: scale must be positive and finite", what);
    CachedArgs a = {};
    a.q = (const bf16_t*)q; a.k_new = (const bf16_t*)k_new; a.v_new = (const bf16_t*)v_new; a.kc = (bf16_t*)k_cache; a.vc = (bf16_t*)v_cache; a.out = (bf16_t*)out;
    a.lengths = lengths; a.batch = batch; a.hq = hq; a.hkv = hkv; a.dim = dim; a.cap = capacity; a.scale = scale;
    a.q_b = q_strides[0]; a.q_h = q_strides[1];
    if (k_new) { a.kn_b = kn_strides[0]; a.kn_h = kn_strides[1]; a.vn_b = vn_strides[0]; a.vn_h = vn_strides[1]; }
    a.k_b = kc_strides[0]; a.k_t = kc_strides[1]; a.k_h = kc_strides[2]; a.v_b = vc_strides[0]; a.v_t = vc_strides[1]; a.v_h = vc_strides[2];
    const int64_t s[12] = {a.q_b, a.q_h, a.kn_b, a.kn_h, a.vn_b, a.vn_h, a.k_b, a.k_t, a.k_h, a.v_b, a.v_t, a.v_h};
    for (int i = 0; i < 12; ++i) GENIE_CHECK_ARG(s[i] >= 0 && s[i] % 8 == 0, "%s: strides must be multiples of 8 elements", what);
    GENIE_CHECK_ARG(a.k_t >= dim && a.v_t >= dim && a.k_t < (1 << 21) && a.v_t < (1 << 21), "%s: a cache row's stride must be between the head width and 2^21 elements", what);
    a.nsplit = cached_splits(batch, hq, hkv, dim, capacity);
    a.hgroups = (hq / hkv + 15) / 16;
    if (a.nsplit > 1) {
        GENIE_CHECK_ARG(ws && ws_floats >= genie_cached_attention_ws_floats(batch, hq, hkv, dim, capacity), "%s: workspace too small", what);
        a.part_o = ws;
        a.part_ml = ws + (int64_t)batch * hq * a.nsplit * dim;
    }
    if (dim <= 32) return cached_dispatch<32>(a, stream);
    if (dim <= 64) return cached_dispatch<64>(a, stream);
    if (dim <= 96) return cached_dispatch<96>(a, stream);
    return cached_dispatch<128>(a, stream);
}
