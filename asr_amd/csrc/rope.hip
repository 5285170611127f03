// asr_qk_norm_rope: RMS norm of the queries and keys of every head, times a learned vector, rotated by the frame's
// position -- one pass over q and k each way.
//
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps);   pairs (p, p + rot/2), p < rot/2:
//   y1 = n1 cos t - n2 sin t,  y2 = n2 cos t + n1 sin t,  t = position * base^(-2p / rot);  the rest of the head: y = n
// backward, gn = the rotation's transpose applied to dy:
//   dw = sum over frames and heads of gn x r,   dx = r (gn w - x r^2 mean(gn w x))
//
// Bound: HBM.  A lane owns V pairs of one head row (both halves, so a rotation never leaves the lane), G = the next power
// of two of D / 2V lanes own a row, and the same lanes walk over HPU heads of the frame: the sine and cosine are
// computed once per frame and pair instead of once per element.  The angle is taken in revolutions in float64 (frames
// of hours of audio: position * frequency has 1e5 revolutions, of which float32 keeps two digits behind the point),
// reduced there and finished in float32.
// Measured: 4 x 4096 frames of 16 + 2 heads of 128 bfloat16 28 us forward (151 MB, 5.4 TB/s), 42 us backward (226 MB, 5.4
// TB/s) and 4 us for the weights' sums; 32 x 374 of 4 + 4 heads of 64 float32 10 and 14.5 us (4.9 and 5.1 TB/s).  A large
// copy reaches 5.15 TB/s.
#include "pieces.h"

struct RopeFreq { double f[64]; };       // frequencies in revolutions per frame, by value: no device table to keep

struct RopeTensor {
    const void *x;                       // (B, T, H, D) with strides
    const void *g;                       // backward: upstream gradient, same shape
    const float *w;
    void *y;                             // forward: output, backward: dx; contiguous (B, T, H, D)
    int64_t xb, xt, xh, gb, gt, gh;
    int H;
};
struct RopeParams {
    RopeTensor t[2];                     // queries, keys
    const int64_t *pos;
    int64_t pos_b;                       // position stride of a batch entry (0: one row for all)
    int64_t ntok;
    int T, D, rot;
    int hpu[2], nhb[2];                  // of each side: head rows per unit of work, units per frame
    int blk[2];                          // workgroups of each side: queries first
    float eps;
    float *part;                         // backward: [blocks][D]
};

// sine and cosine of 2 pi u for |u| <= 1/2: reduced to an eighth of a turn, Taylor to x^9 / x^10 (error below 3e-9)
__device__ __forceinline__ void sincos_rev(float u, float &s, float &c) {
    const float q = rintf(u * 4.f);
    const float x = (u - q * 0.25f) * 6.28318530717958647692f, x2 = x * x;
    const float sp = x + x * x2 * (-1.f / 6 + x2 * (1.f / 120 + x2 * (-1.f / 5040 + x2 * (1.f / 362880))));
    const float cp = 1.f + x2 * (-0.5f + x2 * (1.f / 24 + x2 * (-1.f / 720 + x2 * (1.f / 40320 - x2 * (1.f / 3628800)))));
    const int iq = (int)q;
    const float a = (iq & 1) ? cp : sp, b = (iq & 1) ? sp : cp;
    s = (iq & 2) ? -a : a;
    c = ((iq + 1) & 2) ? -b : b;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
    if (G > 1) v += ASR_DPP(v, 0xB1);            // xor 1
    if (G > 2) v += ASR_DPP(v, 0x4E);            // xor 2
    if (G > 4) v += ASR_DPP(v, 0x141);           // the other quad of eight lanes
    if (G > 8) v += ASR_DPP(v, 0x128);           // the other eight of a row
    if (G > 16) v += __shfl_xor(v, 16, 64);
    if (G > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// what a lane owns of a row: element offsets of its two chunks, and the cosines / sines of one frame
template <int V>
struct RopeLane {
    int lo, hi;
    double f[V];
    bool turn;
    __device__ __forceinline__ void init(const RopeParams &p, const RopeFreq &fr, int l) {
        const int pair = l * V, half = p.rot >> 1;
        turn = pair < half;
        lo = turn ? pair : p.rot + (pair - half);
        hi = turn ? pair + half : lo + ((p.D - p.rot) >> 1);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = turn ? fr.f[pair + i] : 0.0;
    }
    __device__ __forceinline__ void angles(const RopeParams &p, int64_t tok, float (&s)[V], float (&c)[V]) const {
        const int64_t b = tok / p.T, t = tok - b * p.T;
        const double pos = p.pos ? (double)p.pos[b * p.pos_b + t] : (double)t;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double r = pos * f[i];
            sincos_rev((float)(r - rint(r)), s[i], c[i]);
        }
    }
};

template <int DT, int V, int G>
__global__ __launch_bounds__(256) void rope_fwd_kernel(RopeParams p, RopeFreq fr) {
    typedef typename ElemOf<DT>::type E;
    const int side = (int)blockIdx.x >= p.blk[0] ? 1 : 0;
    const RopeTensor &q = p.t[side];
    const int l = threadIdx.x & (G - 1);
    const int64_t unit = (int64_t)(blockIdx.x - (side ? p.blk[0] : 0)) * (256 / G) + threadIdx.x / G;
    const bool on = l * V * 2 < p.D;             // lanes past the row (D / 2V not a power of two) only keep step
    if (unit >= p.ntok * p.nhb[side]) return;    // whole groups leave together
    const int64_t tok = unit / p.nhb[side];
    const int h0 = (int)(unit - tok * p.nhb[side]) * p.hpu[side], h1 = min(h0 + p.hpu[side], q.H);
    RopeLane<V> L;
    L.init(p, fr, on ? l : 0);
    float s[V], c[V];
    L.angles(p, tok, s, c);
    const int64_t b = tok / p.T, t = tok - b * p.T;
    const float inv_d = 1.f / p.D;
    float w1[V], w2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { w1[i] = q.w[L.lo + i]; w2[i] = q.w[L.hi + i]; }
    const E *x = (const E *)q.x + b * q.xb + t * q.xt;
    E *y = (E *)q.y + (tok * q.H) * p.D;
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
        float u[V], v[V];
        load_vec<E, V>(x + h * q.xh + L.lo, u);
        load_vec<E, V>(x + h * q.xh + L.hi, v);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss += u[i] * u[i] + v[i] * v[i];
        const float r = 1.f / sqrtf(group_sum<G>(on ? ss : 0.f) * inv_d + p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float n1 = u[i] * r * w1[i], n2 = v[i] * r * w2[i];
            u[i] = n1 * c[i] - n2 * s[i];
            v[i] = n2 * c[i] + n1 * s[i];
        }
        if (on) {
            store_vec<E, V>(y + h * p.D + L.lo, u);
            store_vec<E, V>(y + h * p.D + L.hi, v);
        }
    }
}

// A workgroup works on one side (half the accumulators and weights in registers: four waves a SIMD instead of two).  The
// weight gradients stay in the lane over all its units; at the end the workgroup's groups are summed through LDS, one partial
// row per workgroup, and rope_dw_kernel adds the rows in a fixed order.
template <int DT, int V, int G>
__global__ __launch_bounds__(256) void rope_bwd_kernel(RopeParams p, RopeFreq fr) {
    typedef typename ElemOf<DT>::type E;
    __shared__ float red[256 * 2 * V];
    const int side = (int)blockIdx.x >= p.blk[0] ? 1 : 0;
    const RopeTensor &q = p.t[side];
    const int l = threadIdx.x & (G - 1);
    const bool on = l * V * 2 < p.D;
    RopeLane<V> L;
    L.init(p, fr, on ? l : 0);
    const float inv_d = 1.f / p.D;
    float dw1[V], dw2[V], w1[V], w2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        dw1[i] = dw2[i] = 0.f;
        w1[i] = q.w[L.lo + i];
        w2[i] = q.w[L.hi + i];
    }
    const int64_t nunit = p.ntok * p.nhb[side], step = (int64_t)p.blk[side] * (256 / G);
    for (int64_t unit = (int64_t)(blockIdx.x - (side ? p.blk[0] : 0)) * (256 / G) + threadIdx.x / G; unit < nunit; unit += step) {
        const int64_t tok = unit / p.nhb[side];
        const int h0 = (int)(unit - tok * p.nhb[side]) * p.hpu[side], h1 = min(h0 + p.hpu[side], q.H);
        float s[V], c[V];
        L.angles(p, tok, s, c);
        const int64_t b = tok / p.T, t = tok - b * p.T;
        const E *x = (const E *)q.x + b * q.xb + t * q.xt;
        const E *g = (const E *)q.g + b * q.gb + t * q.gt;
        E *y = (E *)q.y + (tok * q.H) * p.D;
#pragma unroll 2
        for (int h = h0; h < h1; ++h) {
            float u[V], v[V], gu[V], gv[V];
            load_vec<E, V>(x + h * q.xh + L.lo, u);
            load_vec<E, V>(x + h * q.xh + L.hi, v);
            load_vec<E, V>(g + h * q.gh + L.lo, gu);
            load_vec<E, V>(g + h * q.gh + L.hi, gv);
            float ss = 0.f, sg = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n1 = gu[i] * c[i] + gv[i] * s[i], n2 = gv[i] * c[i] - gu[i] * s[i];
                gu[i] = n1;
                gv[i] = n2;
                ss += u[i] * u[i] + v[i] * v[i];
                sg += n1 * w1[i] * u[i] + n2 * w2[i] * v[i];
            }
            const float r = 1.f / sqrtf(group_sum<G>(on ? ss : 0.f) * inv_d + p.eps);
            const float m = group_sum<G>(on ? sg : 0.f) * inv_d * r * r;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dw1[i] += gu[i] * u[i] * r;
                dw2[i] += gv[i] * v[i] * r;
                u[i] = r * (gu[i] * w1[i] - u[i] * m);
                v[i] = r * (gv[i] * w2[i] - v[i] * m);
            }
            if (on) {
                store_vec<E, V>(y + h * p.D + L.lo, u);
                store_vec<E, V>(y + h * p.D + L.hi, v);
            }
        }
    }
    // red[group][lane][half][i]: column (lane, half, i) of every group at the same offset, one thread a column
#pragma unroll
    for (int i = 0; i < V; ++i) {
        red[threadIdx.x * 2 * V + i] = on ? dw1[i] : 0.f;
        red[threadIdx.x * 2 * V + V + i] = on ? dw2[i] : 0.f;
    }
    __syncthreads();
    if (threadIdx.x < G * 2 * V) {
        const int cl = threadIdx.x / (2 * V), ch = (threadIdx.x / V) & 1, ci = threadIdx.x % V;
        float a = 0.f;
#pragma unroll 8
        for (int k = 0; k < 256 / G; ++k) a += red[k * G * 2 * V + threadIdx.x];
        if (cl * V * 2 < p.D) {
            const int pair = cl * V, half = p.rot >> 1;
            const int lo = pair < half ? pair : p.rot + (pair - half), hi = pair < half ? pair + half : lo + ((p.D - p.rot) >> 1);
            p.part[(int64_t)blockIdx.x * p.D + (ch ? hi : lo) + ci] = a;
        }
    }
}

// dw[col] = sum over a side's workgroups of part[block][col]: 16 columns a workgroup, 64 rows of it in parallel
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float *__restrict__ part, int nq, int nk, int D, float *__restrict__ dwq,
                                                       float *__restrict__ dwk) {
    __shared__ float red[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4, k0 = blockIdx.y ? nq : 0, k1 = blockIdx.y ? nq + nk : nq;
    float a = 0.f;
    if (c < D)
#pragma unroll 8
        for (int k = k0 + r; k < k1; k += 64) a += part[(int64_t)k * D + c];
    red[r][threadIdx.x & 15] = a;
    __syncthreads();
    if (r == 0 && c < D) {
        float s = 0.f;
#pragma unroll 16
        for (int k = 0; k < 64; ++k) s += red[k][threadIdx.x];
        (blockIdx.y ? dwk : dwq)[c] = s;
    }
}

// ------------------------------------------------------------------------------------------------------- host --
// Pairs a lane owns: the widest access of at most 16 bytes that divides both halves of both parts and the alignment.
static int rope_pairs(const asr_rope_args *a, bool bwd) {
    const int es = a->dtype == ASR_T_F32 ? 4 : 2;
    int v = 16 / es;
    const int64_t st[] = {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh};
    const int64_t gs[] = {a->gq_sb, a->gq_st, a->gq_sh, a->gk_sb, a->gk_st, a->gk_sh};
    const void *ptr[] = {a->q, a->k, a->q_out, a->k_out, bwd ? a->gq : nullptr, bwd ? a->gk : nullptr};
    for (; v > 1; v >>= 1) {
        bool ok = (a->rot / 2) % v == 0 && ((a->D - a->rot) / 2) % v == 0;
        for (int64_t s : st) ok = ok && s % v == 0;
        if (bwd) for (int64_t s : gs) ok = ok && s % v == 0;
        for (const void *q : ptr) ok = ok && (uintptr_t)q % (v * es) == 0;
        if (ok) break;
    }
    return v;
}

static int rope_check(const asr_rope_args *a, const char *who) {
    ASR_CHECK_ARG(a && a->q && a->k && a->wq && a->wk && a->q_out && a->k_out, "%s: null pointer", who);
    ASR_CHECK_ARG(a->dtype >= 0 && a->dtype <= 2, "%s: unknown element type", who);
    ASR_CHECK_ARG(a->B > 0 && a->T > 0 && a->H > 0 && a->Hk > 0, "%s: empty shape", who);
    ASR_CHECK_ARG(a->D >= 2 && a->D <= 128 && a->D % 2 == 0, "%s: head width must be even and in [2, 128]", who);
    ASR_CHECK_ARG(a->rot >= 0 && a->rot <= a->D && a->rot % 2 == 0, "%s: rot must be even and in [0, D]", who);
    ASR_CHECK_ARG(a->base > 0.0 && a->eps >= 0.f, "%s: base must be positive, eps not negative", who);
    return ASR_OK;
}

static void rope_fill(const asr_rope_args *a, bool bwd, RopeParams &p, RopeFreq &fr) {
    p.t[0] = RopeTensor{a->q, a->gq, a->wq, a->q_out, a->q_sb, a->q_st, a->q_sh, a->gq_sb, a->gq_st, a->gq_sh, a->H};
    p.t[1] = RopeTensor{a->k, a->gk, a->wk, a->k_out, a->k_sb, a->k_st, a->k_sh, a->gk_sb, a->gk_st, a->gk_sh, a->Hk};
    p.pos = a->pos;
    p.pos_b = a->pos_sb;
    p.ntok = (int64_t)a->B * a->T;
    p.T = a->T;
    p.D = a->D;
    p.rot = a->rot;
    p.eps = a->eps;
    p.part = bwd ? a->ws : nullptr;
    for (int i = 0; i < a->rot / 2; ++i) fr.f[i] = pow(a->base, -2.0 * i / a->rot) / 6.28318530717958647692528676655900577;
    for (int i = a->rot / 2; i < 64; ++i) fr.f[i] = 0.0;
}

// Head rows per unit: all of a frame's on its side (one sine per pair and frame), fewer while the launch has less than 2^17
// lanes of work (a lane then waits on memory, and more of them in flight matter more than the sines).  3 x 777 frames of 6 + 3
// heads of 80, forward / backward: 2^16 6.3 / 7.3 us, 2^17 5.5 / 6.6, 2^18 6.1 / 8.3; 4 x 4096 of 16 + 2 heads of 128,
// backward: 2^17 42 us, 2^20 48.
static void rope_units(RopeParams &p, int G) {
    for (int s = 0; s < 2; ++s) {
        int hpu = p.t[s].H;
        const int Hall = p.t[0].H + p.t[1].H;
        while (hpu > 1 && p.ntok * cdiv(Hall, hpu) * G < (1 << 17)) hpu = (hpu + 1) / 2;
        p.hpu[s] = hpu;
        p.nhb[s] = cdiv(p.t[s].H, hpu);
    }
}

// Backward: eight workgroups a compute unit, twice what run at once (4 x 4096 frames of 16 + 2 heads of 128: 42 us, with as
// many as run at once 45), each side its share by heads
#define ROPE_BWD_BLOCKS 2048
extern "C" int64_t asr_qk_norm_rope_ws_floats(int D) { return (int64_t)(ROPE_BWD_BLOCKS + 2) * D; }

template <int DT, int V, int G>
static int rope_launch(RopeParams &p, const RopeFreq &fr, float *dwq, float *dwk, bool bwd, hipStream_t st) {
    rope_units(p, G);
    int64_t need[2];
    for (int s = 0; s < 2; ++s) need[s] = (p.ntok * p.nhb[s] + 256 / G - 1) / (256 / G);
    ASR_CHECK_ARG(need[0] + need[1] <= 0x7fffffff, "qk_norm_rope: too many frames");
    if (!bwd) {
        p.blk[0] = (int)need[0];
        p.blk[1] = (int)need[1];
        hipLaunchKernelGGL((rope_fwd_kernel<DT, V, G>), dim3((unsigned)(need[0] + need[1])), dim3(256), 0, st, p, fr);
        ASR_CHECK_LAUNCH("rope_fwd_kernel");
        return ASR_OK;
    }
    for (int s = 0; s < 2; ++s) {
        const int64_t share = (int64_t)ROPE_BWD_BLOCKS * p.t[s].H / (p.t[0].H + p.t[1].H) + 1;
        p.blk[s] = (int)(need[s] < share ? need[s] : share);
    }
    hipLaunchKernelGGL((rope_bwd_kernel<DT, V, G>), dim3(p.blk[0] + p.blk[1]), dim3(256), 0, st, p, fr);
    hipLaunchKernelGGL(rope_dw_kernel, dim3(cdiv(p.D, 16), 2), dim3(1024), 0, st, p.part, p.blk[0], p.blk[1], p.D, dwq, dwk);
    ASR_CHECK_LAUNCH("rope_bwd_kernel");
    return ASR_OK;
}

template <int DT, int V>
static int rope_pick_g(RopeParams &p, const RopeFreq &fr, float *dwq, float *dwk, bool bwd, hipStream_t st) {
    const int n = cdiv(p.D, 2 * V);
    if (n <= 1) return rope_launch<DT, V, 1>(p, fr, dwq, dwk, bwd, st);
    if (n <= 2) return rope_launch<DT, V, 2>(p, fr, dwq, dwk, bwd, st);
    if (n <= 4) return rope_launch<DT, V, 4>(p, fr, dwq, dwk, bwd, st);
    if (n <= 8) return rope_launch<DT, V, 8>(p, fr, dwq, dwk, bwd, st);
    if constexpr (V <= 4)
        if (n <= 16) return rope_launch<DT, V, 16>(p, fr, dwq, dwk, bwd, st);
    if constexpr (V <= 2)
        if (n <= 32) return rope_launch<DT, V, 32>(p, fr, dwq, dwk, bwd, st);
    if constexpr (V <= 1) return rope_launch<DT, V, 64>(p, fr, dwq, dwk, bwd, st);
    asr_set_error("qk_norm_rope: no kernel for this width");
    return ASR_ERR_ARG;
}

template <int DT>
static int rope_pick_v(const asr_rope_args *a, RopeParams &p, const RopeFreq &fr, bool bwd, hipStream_t st) {
    switch (rope_pairs(a, bwd)) {
        case 8: if constexpr (DT != ASR_T_F32) return rope_pick_g<DT, 8>(p, fr, a->dwq, a->dwk, bwd, st);
        case 4: return rope_pick_g<DT, 4>(p, fr, a->dwq, a->dwk, bwd, st);
        case 2: return rope_pick_g<DT, 2>(p, fr, a->dwq, a->dwk, bwd, st);
        default: return rope_pick_g<DT, 1>(p, fr, a->dwq, a->dwk, bwd, st);
    }
}

static int rope_run(const asr_rope_args *a, bool bwd, void *stream) {
    RopeParams p;
    RopeFreq fr;
    rope_fill(a, bwd, p, fr);
    switch (a->dtype) {
        case ASR_T_F32: return rope_pick_v<ASR_T_F32>(a, p, fr, bwd, (hipStream_t)stream);
        case ASR_T_BF16: return rope_pick_v<ASR_T_BF16>(a, p, fr, bwd, (hipStream_t)stream);
        default: return rope_pick_v<ASR_T_F16>(a, p, fr, bwd, (hipStream_t)stream);
    }
}

extern "C" int asr_qk_norm_rope_fwd(const asr_rope_args *a, void *stream) {
    ASR_CHECK(rope_check(a, "qk_norm_rope_fwd"));
    return rope_run(a, false, stream);
}

extern "C" int asr_qk_norm_rope_bwd(const asr_rope_args *a, void *stream) {
    ASR_CHECK(rope_check(a, "qk_norm_rope_bwd"));
    ASR_CHECK_ARG(a->gq && a->gk && a->dwq && a->dwk && a->ws, "qk_norm_rope_bwd: null pointer");
    return rope_run(a, true, stream);
}
