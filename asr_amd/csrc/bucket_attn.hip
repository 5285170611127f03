// asr_bucket_attention: softmax attention whose scores carry a learned bias by the bucket of the distance between key and
// query, shared key / value heads, padded batches, causal or not; gradients of q, k, v and of the bias table; a split form
// for a few queries against a long cache.
//
//   S = scale q k^T + table[bucket(j - pos(i))],  P = softmax over the allowed keys (a row without any: zeros),  O = P v
//   dV = P^T dO,  dP = dO v^T,  dS = P (dP - delta),  delta = rowsum(dO O),  dQ = scale dS k,  dK = scale dS^T q,
//   dtable[n] = sum of dS over the pairs in bucket n
//
// The maps are never written.  A wave owns 32 queries (forward, dQ) or 32 keys (dK, dV); the other side streams through LDS.
// Products are v_mfma_f32_32x32x16_bf16 over the pieces of pieces.h.  Orientation: the owned side is the column of the score
// tile, i.e. the lane; a lane then holds 16 scores of ONE query (or key), the row statistics are lane values, and the
// probabilities it holds are already the right-hand operand of the next product (the order of the summed index is the same
// on both operands: slot (half, e) of a 16-step is row 16 c + 8 (e / 4) + 4 half + e % 4, which is how the transposing LDS
// reads deliver the left operand).  Nothing is shuffled between the two products.
//
// Bound: with 16-bit tensors the vector units beside the matrix cores: 64 scores (a register of a wave) cost a fused
// multiply-add, a maximum, a subtraction, an exponential (a quarter-rate instruction), a sum and half a conversion, 34 cycles, and
// 16 matrix cycles at D = 64, 32 at D = 128; a training forward's three pieces of P make that 64 there, the larger side.  So:
// base-2 exponentials with the scale and the bias folded into one multiply-add; the running maximum only moves (and rescales
// the output) when a score exceeds it by 2^8; tiles that need no mask have none; beyond the last bucket edge the bias is one
// number per tile; closer, it is one LDS read at a fixed offset from the lane's distance (a line of biases by distance per head).
//
// Two passes backward (dQ with the table's gradient, dK with dV), each forming S and dP again: 14 D operations a pair
// instead of 10, and no atomics: every sum has a fixed order.
//
// Measured, rates in bf16 matrix operations: bfloat16 2 x 4096 causal, 16 heads of 128 on 2: forward 332 us (0.41 PFLOP/s of
// the formula, 0.83 with the further pieces of P), dQ 349 (0.59; 0.79), dK and dV 460 (0.60); float32 32 x 374, 4 heads of 64, half
// to whole lengths: 44, 64 and 67 us (0.63 to 0.82 PFLOP/s of six products a product over padded maps), packing 18 us a pass at 5.1 TB/s.
#include "pieces.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4a __attribute__((ext_vector_type(4)));
typedef short s16x8a __attribute__((ext_vector_type(8)));

#define LOG2E 1.44269504088896340736f
#define LUT_PAD 64
#define MAX_EDGES 128
#define MAX_REACH 1024
#define PATCH 72                        // words of a patch row: four rows apart is half the banks

// A (B, T, H, D) operand as NP planes of bf16
struct AttnMat {
    const __bf16 *p;
    int64_t sb, st, sh, ps;
};
struct Buckets {
    int nb, nd, first, nedge, causal, R;         // nd: buckets of a direction; R: from this distance on the last one
    int16_t edge[MAX_EDGES];
};
struct AttnParams {
    AttnMat q, k, v, g;
    const float *table;
    const int32_t *lengths, *offset;
    const uint8_t *keep;
    void *out;                                   // (B, Tq, H, D) contiguous
    float *out32, *lse;                          // training: O before rounding (16-bit types), and log2 of the row sums (B, H, Tq)
    const float *delta;
    int B, H, Hk, G, Tq, Tk, D, ntile;
    float scale;
    // backward
    void *dq, *dk, *dv;
    float *tpart, *kvpart;                       // [B * H * q tiles][nb], [gsplit][2][B, Tk, Hk, D]
    int gsplit;
    // few queries
    float *po, *pml;
    const void *kraw, *vraw, *qraw;
    int nsplit;
    Buckets bk;
};

// What a workgroup keeps of the buckets: the edges, and the biases of one head times log2(e)
struct BucketLds {
    float tab[256];
    int16_t edge[MAX_EDGES];
};
__device__ __forceinline__ int bucket_of(const Buckets &b, const int16_t *edge, int r) {
    const int away = b.causal ? max(-r, 0) : abs(r);
    int n = away;
    if (away >= b.first) {                       // edges <= away, by halving
        int lo = 0, hi = b.nedge;
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (edge[m] <= away) lo = m + 1;
            else hi = m;
        }
        n = b.first + lo;
    }
    return n + (!b.causal && r > 0 ? b.nd : 0);
}
// biases by distance -R - PAD .. R + PAD of one head, times log2(e); ends with the line written but not yet visible
__device__ __forceinline__ void fill_lut(float *lut, BucketLds &s, const AttnParams &p, int h) {
    const int R = p.bk.R;
    for (int i = threadIdx.x; i < p.bk.nb; i += 256) s.tab[i] = p.table ? p.table[i * p.H + h] * LOG2E : 0.f;
    if ((int)threadIdx.x < p.bk.nedge) s.edge[threadIdx.x] = p.bk.edge[threadIdx.x];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * (R + LUT_PAD) + 1; i += 256)
        lut[i] = s.tab[bucket_of(p.bk, s.edge, min(max(i - R - LUT_PAD, -R), R))];
}

// An image holds rows of DP bf16 without padding; the 16-byte chunks of a row are permuted by an exclusive or that depends
// on the row, so that both kinds of read are free of bank conflicts: the same chunk of 16 consecutive rows (ds_read_b128,
// 256 B) falls on 16 different sixteenths of the banks, and 64 B of four consecutive rows (the transposing reads of
// two 16-lane groups) on four different quarters.
template <int DP>
__device__ __forceinline__ int swz(int row) {
    return DP == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : DP == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
}
template <int DP>
__device__ __forceinline__ int img_at(int row, int chunk) { return row * 2 * DP + ((chunk ^ swz<DP>(row)) << 4); }
// rows r0 + lane&31, d = 16 ks + 8 half ..+7; r0 is a multiple of 16
template <int DP>
__device__ __forceinline__ bf16x8 frag_rows(const unsigned char *img, int r0, int ks, int lane) {
    const u32x4p v = *reinterpret_cast<const u32x4p *>(img + r0 * 2 * DP + img_at<DP>(lane & 31, ks * 2 + (lane >> 5)));
    return __builtin_bit_cast(bf16x8, v);
}
// transposed: rows d = d0 + lane&31; summed index slot (half, e) = image row r0 + 16 c + 8 (e / 4) + 4 half + e % 4
template <int DP>
__device__ __forceinline__ bf16x8 frag_cols(const unsigned char *img, int r0, int c, int d0, int lane) {
    const int q = 4 * (lane >> 5) + ((lane & 15) >> 2), p = lane & 3, ch = d0 / 8 + 2 * ((lane >> 4) & 1) + (p >> 1);
    const unsigned char *a = img + (r0 + 16 * c) * 2 * DP + 8 * (p & 1);
    typedef __attribute__((address_space(3))) s16x4a *lds_p;
    const s16x4a v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + img_at<DP>(q, ch)));
    const s16x4a v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + img_at<DP>(q + 8, ch)));
    const s16x8a v = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    return __builtin_bit_cast(bf16x8, v);
}
// an owned row's fragments, straight from memory; zero where `on` is false or past D
template <int NP, int DP>
__device__ __forceinline__ void own_rows(bf16x8 (&f)[NP][DP / 16], const AttnMat &m, int64_t b, int64_t h, int64_t row, bool on,
                                         int D, int lane) {
    const __bf16 *a = m.p + b * m.sb + h * m.sh + row * m.st;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
            const int d = 16 * ks + 8 * (lane >> 5);
            u32x4p v = {0u, 0u, 0u, 0u};
            if (on && d < D) v = *reinterpret_cast<const u32x4p *>(a + q * m.ps + d);
            f[q][ks] = __builtin_bit_cast(bf16x8, v);
        }
}

// A tile of ROWS rows of one head on its way into LDS; rows from `n` on, rows that `keep` drops and columns past D are zeros
template <int NP, int DP, int ROWS>
struct RowTile {
    static constexpr int CH = DP / 8, NS = (ROWS * CH + 255) / 256, IMG = ROWS * 2 * DP;
    const __bf16 *p;
    int64_t st, ps;
    u32x4p v[NP][NS];
    unsigned ok, live;                           // live: of row t0 + threadIdx (below ROWS), whether it takes part
    __device__ __forceinline__ void init(const AttnMat &m, int64_t b, int64_t h) {
        p = m.p + b * m.sb + h * m.sh;
        st = m.st;
        ps = m.ps;
    }
    __device__ __forceinline__ void load(int t0, int n, int D, const uint8_t *keep) {
        ok = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int f = threadIdx.x + 256 * i, row = t0 + f / CH, d = (f % CH) * 8;
            const bool in = row < n && d < D;
            const int64_t o = (int64_t)(row < n ? row : n - 1) * st + (d < D ? d : 0);
            if (in && (keep == nullptr || keep[row])) ok |= 1u << i;
#pragma unroll
            for (int q = 0; q < NP; ++q) v[q][i] = *reinterpret_cast<const u32x4p *>(p + q * ps + o);
        }
    }
    __device__ __forceinline__ void load_live(int t0, int n, const uint8_t *keep) {
        const int row = t0 + threadIdx.x;
        live = threadIdx.x < ROWS && row < n && (keep == nullptr || keep[row]) ? 1u : 0u;
    }
    __device__ __forceinline__ void store_live(unsigned char *m) const {
        if (threadIdx.x < ROWS) m[threadIdx.x] = (unsigned char)live;
    }
    __device__ __forceinline__ void store(unsigned char *img) const {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int f = threadIdx.x + 256 * i;
            if (ROWS * CH % 256 != 0 && f >= ROWS * CH) continue;
            const u32x4p z = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int q = 0; q < NP; ++q)
                *reinterpret_cast<u32x4p *>(img + q * IMG + img_at<DP>(f / CH, f % CH)) = (ok >> i) & 1 ? v[q][i] : z;
        }
    }
};

template <int N>
__device__ __forceinline__ void zero16(f32x16 (&a)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[i][r] = 0.f;
}
// t += L R over d: L rows of an image (32 rows from r0), R owned fragments; smallest pieces first.  Two pieces take all four
// products, exact ones: what the fourth adds is 2^-16 of a term, but the table's gradient keeps what differs between the passes
// (float16: its error 6e-6 to 1.1e-5 with three, 3e-7 to 8e-7 with four, for 5 % of the time).
template <int NP, int DP>
__device__ __forceinline__ void dot_rows(f32x16 &t, const unsigned char *img, int imgsz, int r0, const bf16x8 (&own)[NP][DP / 16], int lane) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        bf16x8 a[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) a[q] = frag_rows<DP>(img + q * imgsz, r0, ks, lane);
#pragma unroll
        for (int s = NP == 2 ? 2 : NP - 1; s >= 0; --s)
#pragma unroll
            for (int q = s < NP ? s : NP - 1; q >= (s < NP ? 0 : 1); --q) t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[q], own[s - q][ks], t, 0, 0, 0);
    }
}
// the 16 values a lane holds of a tile as the right operand of the next product, in W pieces
template <int W>
__device__ __forceinline__ void to_operand(bf16x8 (&o)[W][2], const f32x16 &t) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        unsigned w[W][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            unsigned x[W];
            split_pair_finite<W>(t[8 * c + 2 * e], t[8 * c + 2 * e + 1], x);
#pragma unroll
            for (int q = 0; q < W; ++q) w[q][e] = x[q];
        }
#pragma unroll
        for (int q = 0; q < W; ++q) o[q][c] = __builtin_bit_cast(bf16x8, u32x4p{w[q][0], w[q][1], w[q][2], w[q][3]});
    }
}
// acc[d][own] += sum over the tile's 32 rows of image^T times operand
template <int NP, int W, int DP>
__device__ __forceinline__ void dot_cols(f32x16 (&acc)[DP / 32], const unsigned char *img, int imgsz, int r0, const bf16x8 (&o)[W][2], int lane) {
    constexpr int TOP = (NP > W ? NP : W) - 1;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
            bf16x8 a[NP];
#pragma unroll
            for (int q = 0; q < NP; ++q) a[q] = frag_cols<DP>(img + q * imgsz, r0, c, t * 32, lane);
#pragma unroll
            for (int s = TOP; s >= 0; --s)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    if (s - q >= 0 && s - q < W) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[q], o[s - q][c], acc[t], 0, 0, 0);
        }
}
// The same two products in two parts, so that the fragments of one can be read under the other's matrix instructions: with
// one wave a SIMD every read that is waited for right away costs its whole latency (dK and dV of the long bfloat16 case: 41
// such waits a tile, half of its time)
template <int NP, int DP>
struct RowFrags {
    bf16x8 f[NP][DP / 16];
    __device__ __forceinline__ void read(const unsigned char *img, int imgsz, int r0, int lane) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int q = 0; q < NP; ++q) f[q][ks] = frag_rows<DP>(img + q * imgsz, r0, ks, lane);
    }
    __device__ __forceinline__ void dot(f32x16 &t, const bf16x8 (&own)[NP][DP / 16]) const {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int s = NP - 1; s >= 0; --s)
#pragma unroll
                for (int q = s; q >= 0; --q) t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[q][ks], own[s - q][ks], t, 0, 0, 0);
    }
};
template <int NP, int DP>
struct ColFrags {
    bf16x8 f[NP][2][DP / 32];
    __device__ __forceinline__ void read(const unsigned char *img, int imgsz, int r0, int lane) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q) f[q][c][t] = frag_cols<DP>(img + q * imgsz, r0, c, t * 32, lane);
    }
    template <int W>
    __device__ __forceinline__ void dot(f32x16 (&acc)[DP / 32], const bf16x8 (&o)[W][2]) const {
        constexpr int TOP = (NP > W ? NP : W) - 1;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int s = TOP; s >= 0; --s)
#pragma unroll
                for (int q = 0; q < NP; ++q)
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t)
                        if (s - q >= 0 && s - q < W) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[q][c][t], o[s - q][c], acc[t], 0, 0, 0);
    }
};
#define PHASE() __builtin_amdgcn_sched_barrier(0)
__device__ __forceinline__ int row_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// 16 scores of a 32 x 32 tile in base 2: scale and bias added; `first`: distance of register 0 (row 4 half) for this lane,
// dir: +1 where the registers run over keys, -1 where they run over queries.  lo / hi: the tile's extreme distances.
template <int DIR>
__device__ __forceinline__ void add_bias(f32x16 &s, float c, const float *lut, int R, int first, int lo, int hi) {
    if (hi <= -R || lo >= R) {                            // one bucket for the whole tile
        const float b = lut[hi <= -R ? 0 : 2 * (R + LUT_PAD)];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, b);
    } else {
        const float *l = lut + first + R + LUT_PAD;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, l[DIR * (8 * (r >> 2) + (r & 3))]);
    }
}

// four consecutive values of one row of a (B, T, H, D) output
template <typename E>
__device__ __forceinline__ void put4(E *row, int d, int D, float a, float b, float c, float e) {
    const float t[4] = {a, b, c, e};
    if (d + 3 < D && D % 4 == 0) {
        store_vec<E, 4>(row + d, t);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < D) row[d + i] = (E)t[i];
    }
}
template <typename E, int DP>
__device__ __forceinline__ void put_acc(E *row, const f32x16 (&acc)[DP / 32], float f, int D, int half) {
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (t * 32 + 8 * g + 4 * half < D)
                put4<E>(row, t * 32 + 8 * g + 4 * half, D, acc[t][4 * g] * f, acc[t][4 * g + 1] * f, acc[t][4 * g + 2] * f, acc[t][4 * g + 3] * f);
}

template <int NP> struct KeyTile { static constexpr int N = NP == 1 ? 64 : 32; };

// beyond 2^30 from the keys (at most 2^24 of them) nothing changes any more, and sums with frames stay in 32 bits
__device__ __forceinline__ int offset_of(const AttnParams &p, int b) { return p.offset ? min(max(p.offset[b], -(1 << 30)), 1 << 30) : 0; }
__device__ __forceinline__ int keys_of(const AttnParams &p, int b) {
    const int n = p.lengths ? p.lengths[b] : p.Tk;
    return min(max(n, 0), p.Tk);
}

// ------------------------------------------------------------------------------------------------- forward --
// With 16-bit tensors a training forward takes P in three pieces: delta, and with it the sum of a row of dS, is
// as good as O.  Two bfloat16 pieces take 280 us instead of 332 at 2 x 4096 causal, 16 heads of 128, and leave an error of
// 3.8e-6 in dtable instead of 6e-7.  The returned O is rounded to 16 bits once.
// Without gradients bfloat16 takes P in one piece, 8 bits: O is off by 1.33 of its last rounding, training's by 1.0, and two
// pieces would take 256 us instead of 203 at 2 x 4096 causal, 16 heads of 128, 21.6 instead of 18.9 at 32 x 374, 4 heads of 64.
// (Split keys take two: battn_few_kernel.)
template <int DT, int DP, bool TRAIN>
__global__ __launch_bounds__(256, ElemOf<DT>::NP * DP > 192 ? 1 : 2) void battn_fwd_kernel(AttnParams p) {
    constexpr int NP = ElemOf<DT>::NP, W = NP < 3 && TRAIN ? 3 : NP, KT = KeyTile<NP>::N;
    typedef typename ElemOf<DT>::type E;
    typedef RowTile<NP, DP, KT> Tile;
    extern __shared__ __attribute__((aligned(16))) unsigned char pool[];
    __shared__ BucketLds bl;
    __shared__ __attribute__((aligned(4))) unsigned char live[KT];
    unsigned char *ki = pool, *vi = pool + NP * Tile::IMG;
    float *lut = reinterpret_cast<float *>(pool + 2 * NP * Tile::IMG);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int bh = blockIdx.x % (p.B * p.H), b = bh / p.H, h = bh - b * p.H, hk = h / p.G;
    const int q0 = (p.ntile - 1 - (int)(blockIdx.x / (p.B * p.H))) * 128;              // the longest causal rows first
    const int off = offset_of(p, b);
    const int i = q0 + wave * 32 + (lane & 31);
    const int n = keys_of(p, b);
    const int last = off + min(q0 + 127, p.Tq - 1);
    const int kend = p.bk.causal ? min(n, max(last + 1, 0)) : n;
    const uint8_t *keep = p.keep ? p.keep + (int64_t)b * p.Tk : nullptr;
    const int R = p.bk.R;
    bf16x8 qf[NP][DP / 16];
    own_rows<NP, DP>(qf, p.q, b, h, min(i, p.Tq - 1), i < p.Tq, p.D, lane);
    fill_lut(lut, bl, p, h);
    f32x16 o[DP / 32];
    zero16(o);
    float m = -INFINITY, ms = 0.f, l = 0.f;
    const float c = p.scale * LOG2E;
    const int pos = off + i, pmin = off + q0 + wave * 32, pmax = pmin + 31;
    Tile kt, vt;
    kt.init(p.k, b, hk);
    vt.init(p.v, b, hk);
    if (kend > 0) {
        kt.load(0, kend, p.D, keep);
        vt.load(0, kend, p.D, keep);
        kt.load_live(0, kend, keep);
    }
    for (int j0 = 0; j0 < kend; j0 += KT) {
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        kt.store_live(live);
        __syncthreads();
        if (j0 + KT < kend) {
            kt.load(j0 + KT, kend, p.D, keep);
            vt.load(j0 + KT, kend, p.D, keep);
            kt.load_live(j0 + KT, kend, keep);
        }
#pragma unroll 1
        for (int s0 = 0; s0 < KT; s0 += 32) {
            const int j = j0 + s0;
            if (j >= kend || (p.bk.causal && j > pmax)) break;
            f32x16 s[1];
            zero16(s);
            dot_rows<NP, DP>(s[0], ki, Tile::IMG, s0, qf, lane);
            add_bias<1>(s[0], c, lut, R, j + 4 * half - pos, j - pmax, j + 31 - pmin);
            if (j + 32 > kend || keep || (p.bk.causal && j + 31 > pmin)) {
                const int seen = p.bk.causal ? pos - j - 4 * half : 64;                // register rows up to here are not after the query
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const unsigned w = *reinterpret_cast<const unsigned *>(live + s0 + 8 * r4 + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[0][4 * r4 + e] = ((w >> (8 * e)) & 1) && 8 * r4 + e <= seen ? s[0][4 * r4 + e] : -INFINITY;
                }
            }
            float mx = s[0][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[0][r]);
            if (__any(mx > m + 8.f)) {
                mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
                ms = mx == -INFINITY ? 0.f : mx;
                const float a = __builtin_amdgcn_exp2f(m - ms);
                m = mx;
                l *= a;
#pragma unroll
                for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[t][r] *= a;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[0][r] = __builtin_amdgcn_exp2f(s[0][r] - ms);
                l += s[0][r];
            }
            bf16x8 pf[W][2];
            to_operand<W>(pf, s[0]);
            dot_cols<NP, W, DP>(o, vi, Tile::IMG, s0, pf, lane);
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (i >= p.Tq) return;
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);                         // NaN stays NaN
    const int64_t row = ((int64_t)b * p.Tq + i) * p.H + h;
    put_acc<E, DP>((E *)p.out + row * p.D, o, f, p.D, half);
    if (TRAIN) {
        if (NP != 3) put_acc<float, DP>(p.out32 + row * p.D, o, f, p.D, half);
        if (half == 0) p.lse[(int64_t)bh * p.Tq + i] = l > 0.f ? ms + __builtin_amdgcn_logf(l) : (l == 0.f ? INFINITY : l);
    }
}

// ------------------------------------------------------------------------------------------- delta = rowsum(dO O) --
template <int DT>
__global__ __launch_bounds__(256) void battn_delta_kernel(const void *dout, int64_t gb, int64_t gt, int64_t gh, const float *o, float *delta,
                                                          int B, int Tq, int H, int D) {
    typedef typename ElemOf<DT>::type E;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);               // (b, i, h); 16 lanes a row
    const int l = threadIdx.x & 15;
    float s = 0.f;
    if (row < (int64_t)B * Tq * H) {
        const int h = row % H;
        const int64_t bi = row / H, b = bi / Tq, i = bi - b * Tq;
        const E *g = (const E *)dout + b * gb + i * gt + h * gh;
        for (int d = l; d < D; d += 16) s += (float)g[d] * o[row * D + d];
        s = row16_sum(s);
        if (l == 0) delta[(b * H + h) * Tq + i] = s;
    }
}

// ------------------------------------------------------------------------------------- dQ and the table's gradient --
// Sums of dS by distance: 16 keys of a tile at a time go to a patch of LDS of the wave's own, [16][32 + 16 zeros on both
// sides], and lane t adds up the diagonal of distance t - 31 along it (consecutive lanes read consecutive words; the
// zeros stand in for what lies outside), then adds it to the wave's line of sums by distance.  LDS float atomics in its
// place took 250 cycles an instruction: 112 of 302 us of a float32 step at 32 x 374 frames.
// Tiles beyond the last edge add into a register.  At the end the lines are cut into buckets in float64.
// The table's gradient adds up millions of dS that cancel, so what all of them share survives: the matrix instructions round
// their sums down a little more often than up, and every other query's dP is formed negated (float32 at 32 x 374, error of
// dtable against 64 bits: 5.4e-7, without it 2.2e-6).
// Key tiles of 32 where 64 would spill (one piece, D = 128: 302 us against 311 at 2 x 4096 causal, 16 heads).
// With one piece dS goes into dQ in two: a row's dS sum to zero, and what rounding leaves of the sum meets the keys' mean, so
// dQ would be off by up to 1.56 of its own last rounding (2 x 2821 frames, a head of 16; with two 1.0; 349 against 302 us at
// 2 x 4096).  dK and dV take P and dS in one: nothing cancels there, the two roundings add up to 1.41 of one; two pieces would
// cost 562 us against 460.
template <int DT, int DP>
__global__ __launch_bounds__(256, (ElemOf<DT>::NP * DP <= 192 ? 2 : 1)) void battn_dq_kernel(AttnParams p) {
    constexpr int NP = ElemOf<DT>::NP, KT = NP * DP > 64 ? 32 : KeyTile<NP>::N;
    typedef typename ElemOf<DT>::type E;
    typedef RowTile<NP, DP, KT> Tile;
    extern __shared__ __attribute__((aligned(16))) unsigned char pool[];
    __shared__ BucketLds bl;
    __shared__ __attribute__((aligned(4))) unsigned char live[KT];
    const int R = p.bk.R, LN = 2 * (R + LUT_PAD) + 1;
    unsigned char *ki = pool, *vi = pool + NP * Tile::IMG;
    float *lut = reinterpret_cast<float *>(pool + 2 * NP * Tile::IMG);
    float *line = lut + LN;                                                            // 4 lines, 2 x 4 far sums, 4 patches
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int bh = blockIdx.x % (p.B * p.H), b = bh / p.H, h = bh - b * p.H, hk = h / p.G;
    const int qt = p.ntile - 1 - (int)(blockIdx.x / (p.B * p.H)), q0 = qt * 128;
    const int off = offset_of(p, b);
    const int i = q0 + wave * 32 + (lane & 31);
    const bool on = i < p.Tq;
    const int n = keys_of(p, b);
    const int last = off + min(q0 + 127, p.Tq - 1);
    const int kend = p.bk.causal ? min(n, max(last + 1, 0)) : n;
    const uint8_t *keep = p.keep ? p.keep + (int64_t)b * p.Tk : nullptr;
    bf16x8 qf[NP][DP / 16], gf[NP][DP / 16];
    own_rows<NP, DP>(qf, p.q, b, h, min(i, p.Tq - 1), on, p.D, lane);
    own_rows<NP, DP>(gf, p.g, b, h, min(i, p.Tq - 1), on, p.D, lane);
    const float sign = lane & 1 ? -1.f : 1.f;                                          // every other query's dP is formed negated
    if (lane & 1)
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) gf[q][ks] = -gf[q][ks];
    const float lse = on ? p.lse[(int64_t)bh * p.Tq + i] : INFINITY, delta = on ? p.delta[(int64_t)bh * p.Tq + i] : 0.f;
    fill_lut(lut, bl, p, h);
    for (int t = threadIdx.x; t < 4 * LN + 8 + 4 * 16 * PATCH; t += 256) line[t] = 0.f;
    float *mine = line + wave * LN, *patch = line + 4 * LN + 8 + wave * 16 * PATCH;
    f32x16 dq[DP / 32];
    zero16(dq);
    float farl = 0.f, farr = 0.f;
    const float c = p.scale * LOG2E;
    const int pos = off + i, pmin = off + q0 + wave * 32, pmax = pmin + 31;
    Tile kt, vt;
    kt.init(p.k, b, hk);
    vt.init(p.v, b, hk);
    if (kend > 0) {
        kt.load(0, kend, p.D, keep);
        vt.load(0, kend, p.D, keep);
        kt.load_live(0, kend, keep);
    }
    for (int j0 = 0; j0 < kend; j0 += KT) {
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        kt.store_live(live);
        __syncthreads();
        if (j0 + KT < kend) {
            kt.load(j0 + KT, kend, p.D, keep);
            vt.load(j0 + KT, kend, p.D, keep);
            kt.load_live(j0 + KT, kend, keep);
        }
#pragma unroll 1
        for (int s0 = 0; s0 < KT; s0 += 32) {
            const int j = j0 + s0;
            if (j >= kend || (p.bk.causal && j > pmax)) break;
            f32x16 s[2];
            zero16(s);
            dot_rows<NP, DP>(s[0], ki, Tile::IMG, s0, qf, lane);
            dot_rows<NP, DP>(s[1], vi, Tile::IMG, s0, gf, lane);
            const int lo = j - pmax, hi = j + 31 - pmin, first = j + 4 * half - pos;
            add_bias<1>(s[0], c, lut, R, first, lo, hi);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = __builtin_amdgcn_exp2f(s[0][r] - lse) * __builtin_fmaf(sign, s[1][r], -delta);
            if (j + 32 > kend || keep || (p.bk.causal && j + 31 > pmin)) {
                const int seen = p.bk.causal ? pos - j - 4 * half : 64;                // register rows up to here are not after the query
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const unsigned w = *reinterpret_cast<const unsigned *>(live + s0 + 8 * r4 + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[0][4 * r4 + e] = ((w >> (8 * e)) & 1) && 8 * r4 + e <= seen ? s[0][4 * r4 + e] : 0.f;
                }
            }
            if (p.tpart == nullptr) {
                // no table: no sums by distance
            } else if (hi <= -R || lo >= R) {
                float t = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) t += s[0][r];
                if (hi <= -R) farl += t;
                else farr += t;
            } else {
                // lane's diagonal of rows u: distance j + 16 u + t - 31 - (pmin .. ) where t = key row - query column + 31
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    wave_sync();
#pragma unroll
                    for (int r = 0; r < 8; ++r) patch[row_of(r, half) * PATCH + 16 + (lane & 31)] = s[0][8 * u + r];
                    wave_sync();
                    if (lane < 47) {
                        float a = 0.f;
#pragma unroll
                        for (int k = 0; k < 16; ++k) a += patch[k * (PATCH + 1) + 47 - lane];
                        float *d = mine + (j + 16 * u - pmin) + lane - 31 + R + LUT_PAD;
                        *d += a;
                    }
                }
                wave_sync();
            }
            constexpr int W = NP == 1 ? 2 : NP;
            bf16x8 df[W][2];
            to_operand<W>(df, s[0]);
            dot_cols<NP, W, DP>(dq, ki, Tile::IMG, s0, df, lane);
        }
    }
    farl = wave_sum(farl);
    farr = wave_sum(farr);
    if (lane == 0) {
        line[4 * LN + wave] = farl;
        line[4 * LN + 4 + wave] = farr;
    }
    if (on) put_acc<E, DP>((E *)p.dq + (((int64_t)b * p.Tq + i) * p.H + h) * p.D, dq, p.scale, p.D, half);
    if (p.tpart == nullptr) return;
    __syncthreads();
    for (int t = threadIdx.x; t < LN; t += 256) {
        float a = line[t];
#pragma unroll
        for (int u = 1; u < 4; ++u) a += line[u * LN + t];
        line[t] = a;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < p.bk.nb; t += 256) {
        const bool right = !p.bk.causal && t >= p.bk.nd;
        const int k = right ? t - p.bk.nd : t;
        const bool tail = k == p.bk.nd - 1;
        const int lo = max(k <= p.bk.first ? k : (int)bl.edge[k - p.bk.first - 1], right ? 1 : 0);
        const int hi = tail ? R + LUT_PAD + 1 : k < p.bk.first ? k + 1 : (int)bl.edge[k - p.bk.first];
        const float *x = line + R + LUT_PAD;
        double a = 0.0;
#pragma unroll 8
        for (int w = lo; w < hi; ++w) a += x[right ? w : -w];
        if (tail)
#pragma unroll
            for (int u = 0; u < 4; ++u) a += line[4 * LN + (right ? 4 : 0) + u];
        p.tpart[((int64_t)qt * p.B * p.H + bh) * p.bk.nb + t] = (float)a;
    }
}
// dtable[n][h] = sum over utterances and query tiles
__global__ __launch_bounds__(64) void battn_table_kernel(const float *__restrict__ part, float *__restrict__ dt, int B, int H, int ntile, int nb) {
    const int n = blockIdx.x, h = blockIdx.y;
    double a = 0.0;
    for (int t = threadIdx.x; t < B * ntile; t += 64) a += part[((int64_t)t * H + h) * nb + n];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if (threadIdx.x == 0) dt[n * H + h] = (float)a;
}

// ---------------------------------------------------------------------------------------------------- dK and dV --
// Two workgroups a compute unit where 256 registers do: with several pieces that takes loading each tile when it is due (the
// other workgroup hides the wait) and dP behind dV instead of beside S (float32 at 32 x 374, 4 heads of 64: 87 us with one
// workgroup and tiles loaded ahead, 77 with two that spill them, 67).  One piece of D = 128 would still spill (465 -> 660 us).
template <int NP, int DP> struct DkvTwo { static constexpr bool V = NP == 1 ? DP <= 64 : NP * DP <= 192; };
template <int DT, int DP>
__global__ __launch_bounds__(256, (DkvTwo<ElemOf<DT>::NP, DP>::V ? 2 : 1)) void battn_dkv_kernel(AttnParams p) {
    constexpr int NP = ElemOf<DT>::NP, QT = KeyTile<NP>::N;
    typedef typename ElemOf<DT>::type E;
    typedef RowTile<NP, DP, QT> Tile;
    extern __shared__ __attribute__((aligned(16))) unsigned char pool[];
    __shared__ BucketLds bl;
    unsigned char *qi = pool, *gi = pool + NP * Tile::IMG;
    float *stat = reinterpret_cast<float *>(pool + 2 * NP * Tile::IMG);                // lse and delta of the tile's queries
    float *lut = stat + 2 * QT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    // id = (tile, group of heads, utterance and key head): causal, the first keys have most queries and start first
    const int bhk = blockIdx.x % (p.B * p.Hk), b = bhk / p.Hk, hk = bhk - b * p.Hk;
    const int gs = blockIdx.x / (p.B * p.Hk) % p.gsplit, k0 = (int)(blockIdx.x / (p.B * p.Hk) / p.gsplit) * 128;
    const int off = offset_of(p, b);
    const int n = keys_of(p, b);
    const int R = p.bk.R;
    const int jw = k0 + wave * 32, j = jw + (lane & 31);
    const bool on = j < n && (p.keep == nullptr || p.keep[(int64_t)b * p.Tk + j]);
    bf16x8 kf[NP][DP / 16], vf[NP][DP / 16];
    own_rows<NP, DP>(kf, p.k, b, hk, min(j, p.Tk - 1), on, p.D, lane);
    own_rows<NP, DP>(vf, p.v, b, hk, min(j, p.Tk - 1), on, p.D, lane);
    f32x16 dk[DP / 32], dv[DP / 32];
    zero16(dk);
    zero16(dv);
    const float c = p.scale * LOG2E;
    const int i0 = p.bk.causal ? max(0, k0 - off) / QT * QT : 0;                       // the first query that sees the tile's first key
    const int per = (p.G + p.gsplit - 1) / p.gsplit, g0 = gs * per, g1 = min(p.G, g0 + per);
    if (k0 < n)
        for (int gg = g0; gg < g1; ++gg) {
            const int h = hk * p.G + gg;
            const float *lse = p.lse + ((int64_t)b * p.H + h) * p.Tq, *del = p.delta + ((int64_t)b * p.H + h) * p.Tq;
            __syncthreads();
            fill_lut(lut, bl, p, h);
            Tile qt, gt;
            qt.init(p.q, b, h);
            gt.init(p.g, b, h);
            float st = 0.f;                                                            // this thread's lse or delta of the next tile
            auto load_stat = [&](int t0) {
                const int i = t0 + (threadIdx.x & (QT - 1));
                if (threadIdx.x < 2 * QT) st = i >= p.Tq ? (threadIdx.x < QT ? INFINITY : 0.f) : (threadIdx.x < QT ? lse : del)[i];
            };
            constexpr bool AHEAD = NP == 1 || !DkvTwo<NP, DP>::V;
            if (AHEAD && i0 < p.Tq) {
                qt.load(i0, p.Tq, p.D, nullptr);
                gt.load(i0, p.Tq, p.D, nullptr);
                load_stat(i0);
            }
            for (int t0 = i0; t0 < p.Tq; t0 += QT) {
                if (!AHEAD) {
                    qt.load(t0, p.Tq, p.D, nullptr);
                    gt.load(t0, p.Tq, p.D, nullptr);
                    load_stat(t0);
                }
                __syncthreads();
                qt.store(qi);
                gt.store(gi);
                if (threadIdx.x < 2 * QT) stat[threadIdx.x] = st;
                __syncthreads();
                if (AHEAD && t0 + QT < p.Tq) {
                    qt.load(t0 + QT, p.Tq, p.D, nullptr);
                    gt.load(t0 + QT, p.Tq, p.D, nullptr);
                    load_stat(t0 + QT);
                }
                // (a key that is left out collects what it likes in its own column and is stored as zeros)
                auto weigh = [&](f32x16 &s, int s0) {                                  // scores -> probabilities
                    const int pmin = off + t0 + s0;
                    add_bias<-1>(s, c, lut, R, j - (pmin + 4 * half), jw - (pmin + 31), jw + 31 - pmin);
                    if (p.bk.causal && jw + 31 > pmin) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = j <= pmin + row_of(r, half) ? s[r] : -INFINITY;
                    }
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        const f32x4 ls = *reinterpret_cast<const f32x4 *>(stat + s0 + 8 * r4 + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * r4 + e] = __builtin_amdgcn_exp2f(s[4 * r4 + e] - ls[e]);
                    }
                };
                auto slope = [&](f32x16 &dp, const f32x16 &s, int s0) {                // dP -> dS
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        const f32x4 dl = *reinterpret_cast<const f32x4 *>(stat + QT + s0 + 8 * r4 + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dp[4 * r4 + e] = s[4 * r4 + e] * (dp[4 * r4 + e] - dl[e]);
                    }
                };
#pragma unroll 1
                for (int s0 = 0; s0 < QT; s0 += 32) {
                    const int i = t0 + s0, pmax = off + i + 31;
                    if (i >= p.Tq) break;
                    if (jw >= n || (p.bk.causal && jw > pmax)) continue;
                    f32x16 s[1], dp[1];
                    zero16(s);
                    zero16(dp);
                    bf16x8 f[NP][2];
                    if constexpr (NP == 1) {
                        RowFrags<NP, DP> qr, gr;
                        ColFrags<NP, DP> gc, qc;
                        PHASE();
                        qr.read(qi, Tile::IMG, s0, lane);
                        PHASE();
                        gr.read(gi, Tile::IMG, s0, lane);
                        qr.dot(s[0], kf);
                        PHASE();
                        gc.read(gi, Tile::IMG, s0, lane);
                        gr.dot(dp[0], vf);
                        weigh(s[0], s0);
                        to_operand<NP>(f, s[0]);
                        PHASE();
                        qc.read(qi, Tile::IMG, s0, lane);
                        gc.dot(dv, f);
                        slope(dp[0], s[0], s0);
                        to_operand<NP>(f, dp[0]);
                        PHASE();
                        qc.dot(dk, f);
                    } else {
                        dot_rows<NP, DP>(s[0], qi, Tile::IMG, s0, kf, lane);
                        weigh(s[0], s0);
                        to_operand<NP>(f, s[0]);
                        dot_cols<NP, NP, DP>(dv, gi, Tile::IMG, s0, f, lane);
                        dot_rows<NP, DP>(dp[0], gi, Tile::IMG, s0, vf, lane);
                        slope(dp[0], s[0], s0);
                        to_operand<NP>(f, dp[0]);
                        dot_cols<NP, NP, DP>(dk, qi, Tile::IMG, s0, f, lane);
                    }
                }
            }
        }
    if (j >= p.Tk) return;
    const int64_t row = (((int64_t)b * p.Tk + j) * p.Hk + hk) * p.D;
    if (!on) {
        zero16(dk);
        zero16(dv);
    }
    if (p.gsplit > 1) {
        const int64_t sz = (int64_t)p.B * p.Tk * p.Hk * p.D;
        put_acc<float, DP>(p.kvpart + (int64_t)gs * 2 * sz + row, dk, p.scale, p.D, half);
        put_acc<float, DP>(p.kvpart + ((int64_t)gs * 2 + 1) * sz + row, dv, 1.f, p.D, half);
    } else {
        put_acc<E, DP>((E *)p.dk + row, dk, p.scale, p.D, half);
        put_acc<E, DP>((E *)p.dv + row, dv, 1.f, p.D, half);
    }
}
template <int DT>
__global__ __launch_bounds__(256) void battn_kvsum_kernel(const float *__restrict__ part, int64_t sz, int splits, void *dk, void *dv) {
    typedef typename ElemOf<DT>::type E;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * sz; i += (int64_t)gridDim.x * 256) {
        float a = 0.f;
        for (int s = 0; s < splits; ++s) a += part[s * 2 * sz + i];
        if (i < sz) ((E *)dk)[i] = (E)a;
        else ((E *)dv)[i - sz] = (E)a;
    }
}

// ------------------------------------------------------------------------- few queries against many keys, forward --
// The keys of a (utterance, key head) are cut into nsplit runs, one wave each for 32 of the queries; a query's G heads of the
// group are neighbouring columns of the tile, so for single tokens the cache is read once.  A lane loads K as rows (16 bytes of its own key at a time,
// the left operand as it lies) and V as whole lines for the wave's LDS image; the next 32 keys are in flight under the
// current ones: K from where its registers are free, V from where it lies in LDS.  float32 and float16 caches are split into
// pieces in registers.  Only a run that comes near its queries builds the table of buckets, over its own distances.
// A tile's masked keys are one ballot (a byte of the mask a row and element waited for each other: 16 against 12 us for one
// utterance of 150 frames, 4 heads of 40, float16; of these 5 go into the launch, the first loads and the bucket table).
// Bound: the cache's bytes.  16 caches of 4096 to 8192 frames, 16 heads on 2 of 128, bfloat16 (102 MB): 26 us, 3.9 TB/s.
// Registers decide: what spills is reloaded behind the loads in flight and waits for them (36 us with the queries and the LDS
// addresses kept in registers, an index product a load, and a check of D a word).  With one piece the queries therefore lie
// in LDS and the addresses are formed in the loop.  K as whole lines through LDS, like V: 42 against 36 us.
// bfloat16 P goes in as two pieces, 16 bits, so that O is off by its last rounding alone (with one piece by 1.2 to 1.3 of it): the
// matrix cores wait for memory here, and the calls take 0.3 to 0.8 us more (16 caches of 8192: 33.6 against 32.8 us with the join).
// battn_join_kernel joins the runs.
template <int DT, int DP, int MODE>
__global__ __launch_bounds__(64, ElemOf<DT>::NP == 1 ? 2 : 1) void battn_few_kernel(AttnParams p) {
    constexpr bool VEC = MODE > 0, FULL = MODE == 2;                                   // rows of 16-byte words; D = DP
    constexpr bool QL = ElemOf<DT>::NP == 1;                                           // the queries are read from LDS
    constexpr int NP = ElemOf<DT>::NP, PP = NP == 1 ? 2 : NP, IMG = 32 * 2 * DP, CH = DP / 8, NC = DP / 16;
    typedef typename ElemOf<DT>::type E;
    constexpr int W = (int)sizeof(E) / 2;                                              // 16-byte words of eight elements
    extern __shared__ __attribute__((aligned(16))) unsigned char pool[];
    unsigned char *qi = pool + NP * IMG;
    float *tab = reinterpret_cast<float *>(qi + (QL ? IMG : 0));                         // [nb][G] biases of the group's heads
    uint8_t *slot = reinterpret_cast<uint8_t *>(tab + p.bk.nb * p.G);                  // bucket by distance, -R - PAD .. R + PAD
    __shared__ int16_t edge[MAX_EDGES];
    const int lane = threadIdx.x, half = lane >> 5, col = lane & 31;
    const int bhk = blockIdx.x, b = bhk / p.Hk, hk = bhk - b * p.Hk, sp = blockIdx.y;
    const int r0 = blockIdx.z * 32, r1 = min(r0 + 32, p.G * p.Tq) - 1, R = p.bk.R, off = offset_of(p, b);
    const int row = min(r0 + col, r1), g = row % p.G, i = row / p.G, h = hk * p.G + g, pos = off + i;
    const int pmin = off + r0 / p.G, pmax = off + r1 / p.G;
    int n = keys_of(p, b);
    if (p.bk.causal) n = min(n, max(pmax + 1, 0));
    const int run = ((n + p.nsplit - 1) / p.nsplit + 31) / 32 * 32, jb = min(n, sp * run), je = min(n, jb + run);
    const uint8_t *keep = p.keep ? p.keep + (int64_t)b * p.Tk : nullptr;
    // eight elements of a row at d, raw; zeros past D
    struct Raw { u32x4p w[W]; };
    auto raw8 = [&](const E *a, int d) {
        Raw r;
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < W; ++u) r.w[u] = FULL || d < p.D ? reinterpret_cast<const u32x4p *>(a + d)[u] : u32x4p{0u, 0u, 0u, 0u};
        } else {
            E t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = d + e < p.D ? a[d + e] : (E)0.f;
            __builtin_memcpy(&r, t, sizeof(r));
        }
        return r;
    };
    auto pieces8 = [&](const Raw &r, bf16x8 (&o)[NP]) {
        if constexpr (NP == 1) {
            o[0] = __builtin_bit_cast(bf16x8, r.w[0]);
        } else {
            E t[8];
            __builtin_memcpy(t, &r, sizeof(r));
            u32x4p w[NP];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned x[NP];
                split_pair<NP>((float)t[2 * e], (float)t[2 * e + 1], x);
#pragma unroll
                for (int q = 0; q < NP; ++q) w[q][e] = x[q];
            }
#pragma unroll
            for (int q = 0; q < NP; ++q) o[q] = __builtin_bit_cast(bf16x8, w[q]);
        }
    };
    const E *kb = (const E *)p.kraw + b * p.k.sb + (int64_t)hk * p.k.sh, *vb = (const E *)p.vraw + b * p.v.sb + (int64_t)hk * p.v.sh;
    Raw kr[NC], vr[NC];
    bool kept = true;                                                                  // the lane's key of the tile is not masked
    auto load_k = [&](int j0) {
        if (keep) kept = keep[min(j0 + col, je - 1)] != 0;
        const E *k = kb + (int64_t)min(j0 + col, je - 1) * p.k.st;
#pragma unroll
        for (int c = 0; c < NC; ++c) kr[c] = raw8(k, 16 * c + 8 * half);
    };
    auto load_v = [&](int j0) {
        if (64 % CH == 0 && j0 + 32 <= je) {                        // one product of indexes instead of one a load
            const E *v = vb + (int64_t)(j0 + lane / CH) * p.v.st;
#pragma unroll
            for (int c = 0; c < NC; ++c) vr[c] = raw8(v + c * (64 / CH) * p.v.st, lane % CH * 8);
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int f = lane + 64 * c;
                vr[c] = raw8(vb + (int64_t)min(j0 + f / CH, je - 1) * p.v.st, f % CH * 8);
            }
        }
    };
    if (jb < je) {
        load_k(jb);
        load_v(jb);
    }
    bf16x8 qf[QL ? 1 : NP][QL ? 1 : NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        bf16x8 w[NP];
        pieces8(raw8((const E *)p.qraw + b * p.q.sb + (int64_t)i * p.q.st + h * p.q.sh, 16 * c + 8 * half), w);
#pragma unroll
        for (int q = 0; q < NP; ++q)
            if constexpr (QL) *reinterpret_cast<u32x4p *>(qi + q * IMG + img_at<DP>(col, 2 * c + half)) = __builtin_bit_cast(u32x4p, w[q]);
            else qf[q][c] = w[q];
    }
    wave_sync();
    const bool near = !(je - 1 - pmin <= -R || jb - pmax >= R);                        // some key of the run within the last edge
    const float bl = p.table ? p.table[(p.bk.nd - 1) * p.H + h] * LOG2E : 0.f;
    const float br = p.table ? p.table[(p.bk.causal ? 0 : p.bk.nb - 1) * p.H + h] * LOG2E : 0.f;
    if (near) {
        for (int t = lane; t < p.bk.nb * p.G; t += 64) tab[t] = p.table ? p.table[(t / p.G) * p.H + hk * p.G + t % p.G] * LOG2E : 0.f;
        for (int t = lane; t < p.bk.nedge; t += 64) edge[t] = p.bk.edge[t];
        __syncthreads();
        const int lo = max(jb - pmax, -R), hi = min(je + 31 - pmin, R);                // the run's distances
        for (int t = lo + lane; t <= hi; t += 64) slot[t + R + LUT_PAD] = (uint8_t)bucket_of(p.bk, edge, t);
        __syncthreads();
    }
    f32x16 o[DP / 32];
    zero16(o);
    float m = -INFINITY, ms = 0.f, l = 0.f;
    const float c = p.scale * LOG2E;
    for (int j0 = jb; j0 < je; j0 += 32) {
        int ln = lane;                                                                 // LDS addresses are formed in the loop: kept, they spill
        asm volatile("" : "+v"(ln));
        f32x16 s[1];
        zero16(s);
#pragma unroll
        for (int ks = 0; ks < NC; ++ks) {
            bf16x8 w[NP];
            pieces8(kr[ks], w);
#pragma unroll
            for (int t = NP - 1; t >= 0; --t)
#pragma unroll
                for (int q = t; q >= 0; --q) {
                    bf16x8 x;
                    if constexpr (QL) x = frag_rows<DP>(qi + (t - q) * IMG, 0, ks, ln);
                    else x = qf[t - q][ks];
                    s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[q], x, s[0], 0, 0, 0);
                }
        }
        const unsigned live = (unsigned)__ballot(j0 + col < je && kept);
        if (j0 + 32 < je) load_k(j0 + 32);
        wave_sync();
#pragma unroll
        for (int ks = 0; ks < NC; ++ks) {
            bf16x8 w[NP];
            pieces8(vr[ks], w);
            const int f = ln + 64 * ks;
#pragma unroll
            for (int q = 0; q < NP; ++q)
                *reinterpret_cast<u32x4p *>(pool + q * IMG + img_at<DP>(f / CH, f % CH)) =
                    live == 0xffffffffu || (live >> (f / CH) & 1) ? __builtin_bit_cast(u32x4p, w[q]) : u32x4p{0u, 0u, 0u, 0u};
        }
        wave_sync();
        if (j0 + 32 < je) {
            load_v(j0 + 32);
        }
        // (by the tile's last real key, as `near` goes by the run's: a run without a table of buckets has no tile that reads it)
        if (min(j0 + 31, je - 1) - pmin <= -R || j0 - pmax >= R) {
            const float bf = j0 - pmax >= R ? br : bl;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = __builtin_fmaf(s[0][r], c, bf);
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[0][r] = __builtin_fmaf(s[0][r], c, tab[slot[min(max(j0 + row_of(r, half) - pos, -R), R) + R + LUT_PAD] * p.G + g]);
        }
        if (live != 0xffffffffu || (p.bk.causal && j0 + 31 > pmin)) {
            const int seen = p.bk.causal ? pos - j0 - 4 * half : 64;                   // register rows up to here are not after the query
            const unsigned mine = live >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = (mine >> row_of(r, 0) & 1) && row_of(r, 0) <= seen ? s[0][r] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[0][r]);
        if (__any(mx > m + 8.f)) {
            mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            ms = mx == -INFINITY ? 0.f : mx;
            const float a = __builtin_amdgcn_exp2f(m - ms);
            m = mx;
            l *= a;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] *= a;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[0][r] = __builtin_amdgcn_exp2f(s[0][r] - ms);
            l += s[0][r];
        }
        bf16x8 pf[PP][2];
        to_operand<PP>(pf, s[0]);
        dot_cols<NP, PP, DP>(o, pool, IMG, 0, pf, ln);
        wave_sync();
    }
    l += __shfl_xor(l, 32, 64);
    if (r0 + col > r1) return;
    if (p.nsplit == 1) {
        const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        put_acc<E, DP>((E *)p.out + (((int64_t)b * p.Tq + i) * p.H + h) * p.D, o, f, FULL ? DP : p.D, half);
        return;
    }
    const int64_t at = ((int64_t)bhk * p.nsplit + sp) * p.G * p.Tq + row;
    put_acc<float, DP>(p.po + at * p.D, o, 1.f, FULL ? DP : p.D, half);
    if (half == 0) {
        p.pml[2 * at] = m == -INFINITY ? -INFINITY : ms;
        p.pml[2 * at + 1] = l;
    }
}
// One workgroup a row; nsplit <= 64: a lane of each wave has one run's maximum and sum
template <int DT>
__global__ __launch_bounds__(128) void battn_join_kernel(AttnParams p) {
    typedef typename ElemOf<DT>::type E;
    __shared__ float w[64];
    const int rows = p.G * p.Tq, bhk = blockIdx.x / rows, col = blockIdx.x % rows;
    const int b = bhk / p.Hk, hk = bhk - b * p.Hk, g = col % p.G, i = col / p.G, d = threadIdx.x, s = threadIdx.x & 63;
    const int64_t at = (int64_t)bhk * p.nsplit * rows + col;
    const float *po = p.po + at * p.D + min(d, p.D - 1);
    const bool in = s < p.nsplit;
    const float m = in ? p.pml[2 * (at + (int64_t)s * rows)] : -INFINITY, ls = in ? p.pml[2 * (at + (int64_t)s * rows) + 1] : 0.f;
    const float top = wave_max(m), f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
    const float l = wave_sum(f * ls);
    if (threadIdx.x < 64) w[s] = f;
    __syncthreads();
    float a = 0.f;
#pragma unroll 16
    for (int t = 0; t < p.nsplit; ++t) a += w[t] * po[(int64_t)t * rows * p.D];
    if (d < p.D) ((E *)p.out)[(((int64_t)b * p.Tq + i) * p.H + hk * p.G + g) * p.D + d] = (E)(l > 0.f ? a / l : (l == 0.f ? 0.f : l));
}

// ----------------------------------------------------------------------------------- packing into padded planes --
struct AttnPackJob {
    const void *src;
    __bf16 *dst;
    int64_t sb, st, sh, rows;            // rows = B * H * T, laid out (B, H, T, DP)
    int T, H;
    int64_t blk0;
};
struct AttnPack { AttnPackJob j[4]; int n, D, DP; };
template <int DT>
__global__ __launch_bounds__(256) void battn_pack_kernel(AttnPack a) {
    typedef typename ElemOf<DT>::type E;
    constexpr int NP = ElemOf<DT>::NP;
    int k = 0;
    while (k + 1 < a.n && (int64_t)blockIdx.x >= a.j[k + 1].blk0) ++k;
    const AttnPackJob &J = a.j[k];
    const int ch = a.DP / 4;
    const int64_t e = ((int64_t)blockIdx.x - J.blk0) * 256 + threadIdx.x, row = e / ch;
    if (row >= J.rows) return;
    const int d = (int)(e - row * ch) * 4;
    const int64_t bh = row / J.T, t = row - bh * J.T, b = bh / J.H, h = bh - b * J.H;
    const E *s = (const E *)J.src + b * J.sb + t * J.st + h * J.sh + d;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (d + 3 < a.D && (uintptr_t)s % (4 * sizeof(E)) == 0) {
        load_vec<E, 4>(s, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < a.D) v[i] = (float)s[i];
    }
    unsigned lo[NP], hi[NP];
    split_pair<NP>(v[0], v[1], lo);
    split_pair<NP>(v[2], v[3], hi);
#pragma unroll
    for (int q = 0; q < NP; ++q) *reinterpret_cast<u32x2p *>(J.dst + q * J.rows * a.DP + row * a.DP + d) = u32x2p{lo[q], hi[q]};
}

// -------------------------------------------------------------------------------------------------------- host --
static int64_t bup(int64_t v) { return (v + 255) / 256 * 256; }
static int battn_dp(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
static int64_t battn_few_tiles(const asr_bucket_attention_args *a) { return ((int64_t)a->H / a->Hk * a->Tq + 31) / 32; }
// Without gradients the keys are split where there are few queries: one tile of 32 rows a key head, or so few workgroups of
// 128 queries for so many keys that splitting gains more than the smaller tiles cost, and not one for every compute unit: past
// that nothing is left to split, and every 32 queries read all keys for themselves.  us, split against not, at B x T, 4 heads
// of 64: float32 1 x 374 18 / 31, 1 x 1500 57 / 97, 1 x 4096 216 / 246, 1 x 8192 783 / 509, 1 x 16384 2985 / 1543; 4 x 374 35 / 35,
// 8 x 374 47 / 38; bfloat16 1 x 374 13 / 15, 1 x 1500 31 / 43, 1 x 4096 85 / 107, 1 x 8192 274 / 217, 1 x 16384 750 / 532; 1 x 150
// 11 / 9, 4 x 374 21 / 15; one head of 64, 1 x 8192 (64 workgroups) float32 213 / 465.
// (Several tiles: the biases of a group of at most 32 heads lie in LDS.)
static bool battn_few(const asr_bucket_attention_args *a) {
    const int64_t wgs = (int64_t)a->B * a->H * cdiv(a->Tq, 128);
    return !a->train && (battn_few_tiles(a) == 1 || (wgs <= a->Tk / (a->dtype == ASR_T_BF16 ? 24 : 16) && wgs < 256 && a->H / a->Hk <= 32 &&
                                                 battn_few_tiles(a) <= 65535));
}

// Runs of a split cache: about eight waves a compute unit, each run at least 64 keys long (a shorter one spends more on its
// joined row than on its keys)
static int battn_runs(const asr_bucket_attention_args *a) {
    int64_t n = 2048 / ((int64_t)a->B * a->Hk * battn_few_tiles(a));
    if (n > cdiv(a->Tk, 64)) n = cdiv(a->Tk, 64);
    if (n > 64) n = 64;
    return n < 1 ? 1 : (int)n;
}
// bfloat16 tensors whose heads start on the 16-byte grid are operands as they lie
static bool battn_direct(const asr_bucket_attention_args *a, const void *p, int64_t sb, int64_t st, int64_t sh) {
    return a->dtype == ASR_T_BF16 && a->D % 8 == 0 && (uintptr_t)p % 16 == 0 && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
}
struct BattnPlan {
    int NP, DP, ntile, gsplit;
    bool direct[4];
    int64_t off[8], bytes;
};
enum { W_Q, W_K, W_V, W_G, W_DELTA, W_TPART, W_KV };

static void battn_plan(const asr_bucket_attention_args *a, bool bwd, BattnPlan &p) {
    p.NP = a->dtype == ASR_T_F32 ? 3 : a->dtype == ASR_T_F16 ? 2 : 1;
    p.DP = battn_dp(a->D);
    p.ntile = cdiv(a->Tq, 128);
    p.direct[0] = battn_direct(a, a->q, a->q_sb, a->q_st, a->q_sh);
    p.direct[1] = battn_direct(a, a->k, a->k_sb, a->k_st, a->k_sh);
    p.direct[2] = battn_direct(a, a->v, a->v_sb, a->v_st, a->v_sh);
    p.direct[3] = !bwd || battn_direct(a, a->g, a->g_sb, a->g_st, a->g_sh);
    int64_t o = 0;
    auto take = [&](int k, int64_t bytes) {
        p.off[k] = o;
        o += bup(bytes);
    };
    const int64_t e = 2 * p.NP * p.DP, q = (int64_t)a->B * a->H * a->Tq, k = (int64_t)a->B * a->Hk * a->Tk;
    take(W_Q, p.direct[0] ? 0 : q * e);
    take(W_K, p.direct[1] ? 0 : k * e);
    take(W_V, p.direct[2] ? 0 : k * e);
    take(W_G, p.direct[3] ? 0 : q * e);
    p.gsplit = 1;
    if (bwd) {
        take(W_DELTA, q * 4);
        take(W_TPART, (int64_t)a->B * a->H * p.ntile * a->nb * 4);
        // shared key heads: their query heads go to workgroups of their own until there are two for each compute unit
        const int G = a->H / a->Hk;
        while (p.gsplit < G && (int64_t)p.gsplit * a->B * a->Hk * cdiv(a->Tk, 128) < 512) p.gsplit *= 2;
        if (p.gsplit > G) p.gsplit = G;
        take(W_KV, p.gsplit > 1 ? (int64_t)p.gsplit * 2 * k * a->D * 4 : 0);
    }
    p.bytes = o;
}

static int battn_check(const asr_bucket_attention_args *a, const char *who, bool ptrs) {
    ASR_CHECK_ARG(a, "%s: null pointer", who);
    ASR_CHECK_ARG(a->dtype >= 0 && a->dtype <= 2, "%s: unknown element type", who);
    ASR_CHECK_ARG(a->B > 0 && a->Tq > 0 && a->Tk > 0 && a->H > 0 && a->Hk > 0, "%s: empty shape", who);
    ASR_CHECK_ARG(a->H % a->Hk == 0, "%s: the query heads must be a multiple of the key heads", who);
    ASR_CHECK_ARG(a->D >= 1 && a->D <= 128, "%s: head width must be in [1, 128]", who);
    ASR_CHECK_ARG(a->Tq <= (1 << 24) && a->Tk <= (1 << 24), "%s: at most 2^24 frames", who);
    ASR_CHECK_ARG((int64_t)a->B * a->H * cdiv(a->Tq, 128) < (1ll << 31) && (int64_t)a->B * a->H * cdiv(a->Tk, 128) < (1ll << 31) &&
                      (int64_t)a->B * a->H <= (1 << 20), "%s: too many rows", who);
    ASR_CHECK_ARG(a->nb >= 2 && a->nb <= 256 && (a->causal || (a->nb >= 4 && a->nb % 2 == 0)),
                  "%s: 2 to 256 buckets, an even number of at least 4 where keys may follow the query", who);
    const int nd = a->causal ? a->nb : a->nb / 2, first = nd / 2;
    ASR_CHECK_ARG(a->edges_host || nd - first - 1 == 0, "%s: null pointer", who);
    int prev = first;
    for (int i = 0; i < nd - first - 1; ++i) {
        ASR_CHECK_ARG(a->edges_host[i] >= prev && a->edges_host[i] <= MAX_REACH, "%s: bucket edges must not fall, and stay within %d", who, MAX_REACH);
        prev = a->edges_host[i];
    }
    if (ptrs) ASR_CHECK_ARG(a->q && a->k && a->v, "%s: null pointer", who);
    return ASR_OK;
}

static void battn_fill(const asr_bucket_attention_args *a, const BattnPlan &pl, AttnParams &p) {
    p = AttnParams{};
    char *ws = (char *)a->ws;
    const int64_t qr = (int64_t)a->B * a->H * a->Tq, kr = (int64_t)a->B * a->Hk * a->Tk;
    auto mat = [&](int k, const void *src, int64_t sb, int64_t st, int64_t sh, int H, int T, int64_t rows) {
        return pl.direct[k] ? AttnMat{(const __bf16 *)src, sb, st, sh, 0}
                            : AttnMat{(const __bf16 *)(ws + pl.off[k]), (int64_t)H * T * pl.DP, pl.DP, (int64_t)T * pl.DP, rows * pl.DP};
    };
    p.q = mat(0, a->q, a->q_sb, a->q_st, a->q_sh, a->H, a->Tq, qr);
    p.k = mat(1, a->k, a->k_sb, a->k_st, a->k_sh, a->Hk, a->Tk, kr);
    p.v = mat(2, a->v, a->v_sb, a->v_st, a->v_sh, a->Hk, a->Tk, kr);
    p.g = mat(3, a->g, a->g_sb, a->g_st, a->g_sh, a->H, a->Tq, qr);
    p.table = a->table;
    p.lengths = a->lengths;
    p.offset = a->offset;
    p.keep = a->keep;
    p.out = a->out;
    p.out32 = a->out32;
    p.lse = a->lse;
    p.B = a->B;
    p.H = a->H;
    p.Hk = a->Hk;
    p.G = a->H / a->Hk;
    p.Tq = a->Tq;
    p.Tk = a->Tk;
    // packed planes are padded to DP with zeros; an operand as it lies is zero-filled past D on the way
    p.D = a->D;
    p.ntile = pl.ntile;
    p.scale = a->scale;
    p.dq = a->dq;
    p.dk = a->dk;
    p.dv = a->dv;
    p.gsplit = pl.gsplit;
    p.bk.nb = a->nb;
    p.bk.causal = a->causal != 0;
    p.bk.nd = a->causal ? a->nb : a->nb / 2;
    p.bk.first = p.bk.nd / 2;
    p.bk.nedge = p.bk.nd - p.bk.first - 1;
    for (int i = 0; i < p.bk.nedge; ++i) p.bk.edge[i] = (int16_t)a->edges_host[i];
    p.bk.R = p.bk.nedge ? a->edges_host[p.bk.nedge - 1] : p.bk.first;
    if (p.bk.R < 1) p.bk.R = 1;
}

template <int DT>
static int battn_pack(const asr_bucket_attention_args *a, const BattnPlan &pl, bool bwd, hipStream_t st) {
    AttnPack j;
    j.n = 0;
    j.D = a->D;
    j.DP = pl.DP;
    int64_t blocks = 0;
    const void *src[4] = {a->q, a->k, a->v, a->g};
    const int64_t s[4][3] = {{a->q_sb, a->q_st, a->q_sh}, {a->k_sb, a->k_st, a->k_sh}, {a->v_sb, a->v_st, a->v_sh}, {a->g_sb, a->g_st, a->g_sh}};
    for (int k = 0; k < (bwd ? 4 : 3); ++k) {
        if (pl.direct[k]) continue;
        const int H = k == 1 || k == 2 ? a->Hk : a->H, T = k == 1 || k == 2 ? a->Tk : a->Tq;
        const int64_t rows = (int64_t)a->B * H * T;
        j.j[j.n++] = AttnPackJob{src[k], (__bf16 *)((char *)a->ws + pl.off[k]), s[k][0], s[k][1], s[k][2], rows, T, H, blocks};
        blocks += (rows * (pl.DP / 4) + 255) / 256;
    }
    if (!j.n) return ASR_OK;
    ASR_CHECK_ARG(blocks < (1ll << 31), "bucket_attention: too many rows");
    hipLaunchKernelGGL((battn_pack_kernel<DT>), dim3((unsigned)blocks), dim3(256), 0, st, j);
    ASR_CHECK_LAUNCH("battn_pack_kernel");
    return ASR_OK;
}

template <typename K>
static int battn_lds(K kernel, size_t bytes, const char *who) {
    ASR_CHECK_ARG(bytes <= 160 * 1024, "%s: %zu bytes of LDS", who, bytes);
    if (bytes > 64 * 1024) ASR_CHECK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return ASR_OK;
}

template <int DT, int DP>
static int battn_fwd(const asr_bucket_attention_args *a, hipStream_t st) {
    constexpr int NP = ElemOf<DT>::NP, KT = KeyTile<NP>::N;
    AttnParams p;
    BattnPlan pl;
    battn_plan(a, false, pl);
    battn_fill(a, pl, p);
    if (battn_few(a)) {
        p.q.sb = a->q_sb; p.q.st = a->q_st; p.q.sh = a->q_sh;
        p.k.sb = a->k_sb; p.k.st = a->k_st; p.k.sh = a->k_sh;
        p.v.sb = a->v_sb; p.v.st = a->v_st; p.v.sh = a->v_sh;
        p.qraw = a->q;
        p.kraw = a->k;
        p.vraw = a->v;
        const int es = DT == ASR_T_F32 ? 4 : 2, al = 16 / es;
        bool vec = a->D % 8 == 0;
        for (int64_t s : {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh}) vec = vec && s % al == 0;
        for (const void *x : {a->q, a->k, a->v}) vec = vec && (uintptr_t)x % 16 == 0;
        p.nsplit = battn_runs(a);
        const int64_t rows = (int64_t)p.G * p.Tq * a->B * a->Hk;
        p.po = (float *)a->ws;
        p.pml = p.po + rows * p.nsplit * a->D;
        const size_t lds = (NP == 1 ? 2 : NP) * 32 * 2 * DP + sizeof(float) * p.bk.nb * p.G + (2 * (p.bk.R + LUT_PAD) + 1);
        const auto few = !vec ? battn_few_kernel<DT, DP, 0> : a->D < DP ? battn_few_kernel<DT, DP, 1> : battn_few_kernel<DT, DP, 2>;
        ASR_CHECK(battn_lds(few, lds, "bucket_attention_fwd"));
        hipLaunchKernelGGL(few, dim3(a->B * a->Hk, p.nsplit, (unsigned)battn_few_tiles(a)), dim3(64), lds, st, p);
        if (p.nsplit > 1) hipLaunchKernelGGL((battn_join_kernel<DT>), dim3((unsigned)rows), dim3(128), 0, st, p);
        ASR_CHECK_LAUNCH("battn_few_kernel");
        return ASR_OK;
    }
    ASR_CHECK(battn_pack<DT>(a, pl, false, st));
    const size_t lds = 2 * NP * RowTile<NP, DP, KT>::IMG + sizeof(float) * (2 * (p.bk.R + LUT_PAD) + 1);
    const dim3 grid((unsigned)(a->B * a->H) * pl.ntile);
    if (a->train) {
        ASR_CHECK(battn_lds(battn_fwd_kernel<DT, DP, true>, lds, "bucket_attention_fwd"));
        hipLaunchKernelGGL((battn_fwd_kernel<DT, DP, true>), grid, dim3(256), lds, st, p);
    } else {
        ASR_CHECK(battn_lds(battn_fwd_kernel<DT, DP, false>, lds, "bucket_attention_fwd"));
        hipLaunchKernelGGL((battn_fwd_kernel<DT, DP, false>), grid, dim3(256), lds, st, p);
    }
    ASR_CHECK_LAUNCH("battn_fwd_kernel");
    return ASR_OK;
}

template <int DT, int DP>
static int battn_bwd(const asr_bucket_attention_args *a, hipStream_t st) {
    constexpr int NP = ElemOf<DT>::NP, KT = KeyTile<NP>::N;
    AttnParams p;
    BattnPlan pl;
    battn_plan(a, true, pl);
    battn_fill(a, pl, p);
    char *ws = (char *)a->ws;
    float *delta = (float *)(ws + pl.off[W_DELTA]);
    p.delta = delta;
    p.tpart = a->table ? (float *)(ws + pl.off[W_TPART]) : nullptr;
    p.kvpart = (float *)(ws + pl.off[W_KV]);
    ASR_CHECK(battn_pack<DT>(a, pl, true, st));
    const int64_t rows = (int64_t)a->B * a->Tq * a->H;
    hipLaunchKernelGGL((battn_delta_kernel<DT>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a->g, a->g_sb, a->g_st, a->g_sh,
                       DT == ASR_T_F32 ? (const float *)a->out : a->out32, delta, a->B, a->Tq, a->H, a->D);
    ASR_CHECK_LAUNCH("battn_delta_kernel");
    const size_t img = 2 * NP * RowTile<NP, DP, KT>::IMG, line = 2 * (p.bk.R + LUT_PAD) + 1;
    const size_t lds_q = img + sizeof(float) * (5 * line + 8 + 4 * 16 * PATCH), lds_k = img + sizeof(float) * (2 * KT + line);
    ASR_CHECK(battn_lds(battn_dq_kernel<DT, DP>, lds_q, "bucket_attention_bwd"));
    hipLaunchKernelGGL((battn_dq_kernel<DT, DP>), dim3((unsigned)(a->B * a->H) * pl.ntile), dim3(256), lds_q, st, p);
    ASR_CHECK_LAUNCH("battn_dq_kernel");
    if (p.tpart) hipLaunchKernelGGL(battn_table_kernel, dim3(a->nb, a->H), dim3(64), 0, st, p.tpart, a->dtable, a->B, a->H, pl.ntile, a->nb);
    ASR_CHECK(battn_lds(battn_dkv_kernel<DT, DP>, lds_k, "bucket_attention_bwd"));
    hipLaunchKernelGGL((battn_dkv_kernel<DT, DP>), dim3((unsigned)(a->B * a->Hk) * cdiv(a->Tk, 128) * pl.gsplit), dim3(256), lds_k, st, p);
    ASR_CHECK_LAUNCH("battn_dkv_kernel");
    if (pl.gsplit > 1) {
        const int64_t sz = (int64_t)a->B * a->Tk * a->Hk * a->D, nb = (2 * sz + 255) / 256;
        hipLaunchKernelGGL((battn_kvsum_kernel<DT>), dim3((unsigned)(nb < 8192 ? nb : 8192)), dim3(256), 0, st, p.kvpart, sz, pl.gsplit, a->dk, a->dv);
        ASR_CHECK_LAUNCH("battn_kvsum_kernel");
    }
    return ASR_OK;
}

template <int DT>
static int battn_run(const asr_bucket_attention_args *a, bool bwd, hipStream_t st) {
    switch (battn_dp(a->D)) {
        case 32: return bwd ? battn_bwd<DT, 32>(a, st) : battn_fwd<DT, 32>(a, st);
        case 64: return bwd ? battn_bwd<DT, 64>(a, st) : battn_fwd<DT, 64>(a, st);
        case 96: return bwd ? battn_bwd<DT, 96>(a, st) : battn_fwd<DT, 96>(a, st);
        default: return bwd ? battn_bwd<DT, 128>(a, st) : battn_fwd<DT, 128>(a, st);
    }
}
static int battn_any(const asr_bucket_attention_args *a, bool bwd, void *stream) {
    switch (a->dtype) {
        case ASR_T_F32: return battn_run<ASR_T_F32>(a, bwd, (hipStream_t)stream);
        case ASR_T_BF16: return battn_run<ASR_T_BF16>(a, bwd, (hipStream_t)stream);
        default: return battn_run<ASR_T_F16>(a, bwd, (hipStream_t)stream);
    }
}

extern "C" int64_t asr_bucket_attention_ws_bytes(const asr_bucket_attention_args *a, int backward) {
    if (battn_check(a, "bucket_attention_ws_bytes", false) != ASR_OK) return -1;
    if (!backward && battn_few(a)) {
        const int n = battn_runs(a);
        return n > 1 ? bup((int64_t)a->B * a->H * a->Tq * n * (a->D + 2) * 4) : 0;
    }
    BattnPlan p;
    battn_plan(a, backward != 0, p);
    return p.bytes;
}
extern "C" int asr_bucket_attention_fwd(const asr_bucket_attention_args *a, void *stream) {
    ASR_CHECK(battn_check(a, "bucket_attention_fwd", true));
    ASR_CHECK_ARG(a->out && (!a->train || (a->lse && (a->out32 || a->dtype == ASR_T_F32))), "bucket_attention_fwd: null pointer");
    ASR_CHECK_ARG(a->ws || asr_bucket_attention_ws_bytes(a, 0) == 0, "bucket_attention_fwd: null pointer");
    return battn_any(a, false, stream);
}
extern "C" int asr_bucket_attention_bwd(const asr_bucket_attention_args *a, void *stream) {
    ASR_CHECK(battn_check(a, "bucket_attention_bwd", true));
    ASR_CHECK_ARG(a->g && a->lse && a->dq && a->dk && a->dv && (a->dtable || !a->table) && a->ws && (a->dtype == ASR_T_F32 ? a->out != nullptr : a->out32 != nullptr),
                  "bucket_attention_bwd: null pointer");
    return battn_any(a, true, stream);
}
