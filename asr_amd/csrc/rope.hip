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
    int T, D, rot, hpu, nhb;             // hpu: head rows per unit of work, nhb: units per frame
    float eps;
    float *part;                         // backward: [blocks][2][D]
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
    const int l = threadIdx.x & (G - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool on = l * V * 2 < p.D;             // lanes past the row (D / 2V not a power of two) only keep step
    if (unit >= p.ntok * p.nhb) return;          // whole groups leave together
    const int64_t tok = unit / p.nhb;
    const int h0 = (int)(unit - tok * p.nhb) * p.hpu, Hall = p.t[0].H + p.t[1].H, h1 = min(h0 + p.hpu, Hall);
    RopeLane<V> L;
    L.init(p, fr, on ? l : 0);
    float s[V], c[V];
    L.angles(p, tok, s, c);
    const int64_t b = tok / p.T, t = tok - b * p.T;
    const float inv_d = 1.f / p.D;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const RopeTensor &q = p.t[side];
        const int a0 = max(h0 - (side ? p.t[0].H : 0), 0), a1 = min(h1 - (side ? p.t[0].H : 0), q.H);
        if (a0 >= a1) continue;
        float w1[V], w2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { w1[i] = q.w[L.lo + i]; w2[i] = q.w[L.hi + i]; }
        const E *x = (const E *)q.x + b * q.xb + t * q.xt;
        E *y = (E *)q.y + (tok * q.H) * p.D;
#pragma unroll 4
        for (int h = a0; h < a1; ++h) {
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
}

// The weight gradients stay in the lane over all its units and are summed over the block's groups at the end, one
// partial row per block; rope_dw_kernel adds the rows in a fixed order.
template <int DT, int V, int G>
__global__ __launch_bounds__(256) void rope_bwd_kernel(RopeParams p, RopeFreq fr) {
    typedef typename ElemOf<DT>::type E;
    __shared__ float red[256 * 2 * V];
    const int l = threadIdx.x & (G - 1);
    const bool on = l * V * 2 < p.D;
    RopeLane<V> L;
    L.init(p, fr, on ? l : 0);
    const float inv_d = 1.f / p.D;
    float dw[2][2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) dw[0][0][i] = dw[0][1][i] = dw[1][0][i] = dw[1][1][i] = 0.f;
    float w[2][2][V];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int i = 0; i < V; ++i) { w[side][0][i] = p.t[side].w[L.lo + i]; w[side][1][i] = p.t[side].w[L.hi + i]; }
    const int64_t nunit = p.ntok * p.nhb;
    const int Hall = p.t[0].H + p.t[1].H;
    for (int64_t unit = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; unit < nunit; unit += (int64_t)gridDim.x * (256 / G)) {
        const int64_t tok = unit / p.nhb;
        const int h0 = (int)(unit - tok * p.nhb) * p.hpu, h1 = min(h0 + p.hpu, Hall);
        float s[V], c[V];
        L.angles(p, tok, s, c);
        const int64_t b = tok / p.T, t = tok - b * p.T;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const RopeTensor &q = p.t[side];
            const int a0 = max(h0 - (side ? p.t[0].H : 0), 0), a1 = min(h1 - (side ? p.t[0].H : 0), q.H);
            const E *x = (const E *)q.x + b * q.xb + t * q.xt;
            const E *g = (const E *)q.g + b * q.gb + t * q.gt;
            E *y = (E *)q.y + (tok * q.H) * p.D;
#pragma unroll 2
            for (int h = a0; h < a1; ++h) {
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
                    sg += n1 * w[side][0][i] * u[i] + n2 * w[side][1][i] * v[i];
                }
                const float r = 1.f / sqrtf(group_sum<G>(on ? ss : 0.f) * inv_d + p.eps);
                const float m = group_sum<G>(on ? sg : 0.f) * inv_d * r * r;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dw[side][0][i] += gu[i] * u[i] * r;
                    dw[side][1][i] += gv[i] * v[i] * r;
                    u[i] = r * (gu[i] * w[side][0][i] - u[i] * m);
                    v[i] = r * (gv[i] * w[side][1][i] - v[i] * m);
                }
                if (on) {
                    store_vec<E, V>(y + h * p.D + L.lo, u);
                    store_vec<E, V>(y + h * p.D + L.hi, v);
                }
            }
        }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[threadIdx.x * 2 * V + i] = dw[side][0][i];
            red[threadIdx.x * 2 * V + V + i] = dw[side][1][i];
        }
        __syncthreads();
        if (threadIdx.x < G && on) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a = 0.f, e = 0.f;
                for (int k = threadIdx.x; k < 256; k += G) { a += red[k * 2 * V + i]; e += red[k * 2 * V + V + i]; }
                float *out = p.part + ((int64_t)blockIdx.x * 2 + side) * p.D;
                out[L.lo + i] = a;
                out[L.hi + i] = e;
            }
        }
    }
}

// dw[side][col] = sum over blocks of part[block][side][col]: 16 columns a block, 16 rows of it in parallel
__global__ __launch_bounds__(256) void rope_dw_kernel(const float *__restrict__ part, int nblk, int D, float *__restrict__ dwq,
                                                      float *__restrict__ dwk) {
    __shared__ float red[16][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    float a = 0.f;
    if (c < 2 * D)
        for (int k = r; k < nblk; k += 16) a += part[(int64_t)k * 2 * D + c];
    red[r][threadIdx.x & 15] = a;
    __syncthreads();
    if (r == 0 && c < 2 * D) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += red[k][threadIdx.x];
        if (c < D) dwq[c] = s;
        else dwk[c - D] = s;
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

// Head rows per unit: all of a frame's (one sine per pair and frame), fewer while the launch has less than 2^18 lanes of
// work (a lane then waits on memory, and more of them in flight matter more than the sines).
static void rope_units(RopeParams &p, int G) {
    const int Hall = p.t[0].H + p.t[1].H;
    int hpu = Hall;
    while (hpu > 1 && p.ntok * cdiv(Hall, hpu) * G < (1 << 18)) hpu = (hpu + 1) / 2;
    p.hpu = hpu;
    p.nhb = cdiv(Hall, hpu);
}

#define ROPE_BWD_BLOCKS 1024
extern "C" int64_t asr_qk_norm_rope_ws_floats(int D) { return (int64_t)ROPE_BWD_BLOCKS * 2 * D; }

template <int DT, int V, int G>
static int rope_launch(RopeParams &p, const RopeFreq &fr, float *dwq, float *dwk, bool bwd, hipStream_t st) {
    rope_units(p, G);
    const int64_t blocks = (p.ntok * p.nhb + 256 / G - 1) / (256 / G);
    ASR_CHECK_ARG(blocks <= 0x7fffffff, "qk_norm_rope: too many frames");
    if (!bwd) {
        hipLaunchKernelGGL((rope_fwd_kernel<DT, V, G>), dim3((unsigned)blocks), dim3(256), 0, st, p, fr);
        ASR_CHECK_LAUNCH("rope_fwd_kernel");
        return ASR_OK;
    }
    const int nb = blocks < ROPE_BWD_BLOCKS ? (int)blocks : ROPE_BWD_BLOCKS;
    hipLaunchKernelGGL((rope_bwd_kernel<DT, V, G>), dim3(nb), dim3(256), 0, st, p, fr);
    hipLaunchKernelGGL(rope_dw_kernel, dim3(cdiv(2 * p.D, 16)), dim3(256), 0, st, p.part, nb, p.D, dwq, dwk);
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
