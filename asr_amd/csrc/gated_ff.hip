// asr_gated_ff: y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradients; x (M,d), Wg / Wu (f,d), Wd (n,f).
//
// forward   1  a, b = x Wg^T, x Wu^T of one tile, h = act(a) b in the epilogue                (gff_gate_kernel)
//           2  y = h Wd^T                                                                      (gff_nt_kernel)
// backward  1  a, b again and dh = dy Wd of one tile, epilogue: h, da = dh b act'(a), db = dh act(a)
//           2  dx = [da db] [Wg; Wu]                                                           (gff_nt_kernel)
//           3  dWg, dWu = [da db]^T x,  dWd = dy^T h                                           (gff_tn_kernel, split over M)
// Nothing but x is kept for the backward: computing a and b again costs 4 M d f operations of 22 and saves writing and
// reading two M x f arrays each way; it also keeps act' on unrounded a and b.  h, da and db are rounded once, each by
// itself, because the next product reads them as matrix operands (half a step relative to the value: bfloat16 2^-8, one piece of
// pieces.h, which makes the outputs' error 1.4 of their own rounding; float16 2^-16, two; float32 2^-24, three).
//
// Gate and up columns are interleaved by 32, so that a wave holds a and b of the same elements; products are
// v_mfma_f32_32x32x16_bf16 over tiles of 256 rows and eight waves where there are enough of them (the tiles of each product
// stand at its launch), operands staged through registers into two LDS images.
// Bound: the LDS with one piece, whose reads take as long as the matrix work; the matrix cores with more, and in the gate
// kernel the stores behind each tile.  Measured, rates in bf16 matrix operations (a library product of the size: 1.2 PFLOP/s):
//   bfloat16 8192 x 1024 x 4096    gate 163 us (0.84 PFLOP/s), backward 275 (0.75), y and dx 108 each on average (0.95),
//                                  weight gradients 124 each on average (0.83)
//   float32 11968 x 256 x 2048     gate 178 (0.85), backward 329 (0.69; without its 441 MB of stores 261), y and dx 133 (0.85),
//                                  weight gradients 107 (1.06)
//   float16 3000 x 1024 x 4096     a training call 739 us, without gradients 173 (bfloat16: training 392); with operands of
//                                  the gate kernel in pieces too 918 and 238
//   bfloat16 8 x 1024 x 4096       8.3 + 5.2 + 2.3 us in three launches: 25 MB of weights at 1.6 TB/s, three waits long
// Rows and columns beyond the matrix are read from its last row (clamped) and masked in the epilogues; the arrays h, da, db
// are padded to whole tiles with zeros, which is what the products over them read past the end.
#include <type_traits>
#include "pieces.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4g __attribute__((ext_vector_type(4)));
typedef short s16x8g __attribute__((ext_vector_type(8)));

enum { GFF_SWISH = 0, GFF_GELU = 1 };

// float16 operands of the gate kernel (x, Wg, Wu, dy, Wd) go into v_mfma_f32_32x32x16_f16 as they lie: one exact product, like
// bfloat16 (F16_AS_IS).  What it forms from them, h, da and db, may leave the range of float16 where y and the gradients do not,
// and one large row of x or dy must not cost the others bits, so the products over those take two bf16 pieces a value, three
// products: 16 bits of every value by itself, over the range of float32.  (One power of two for a whole h, from the largest
// row norms, would keep single products, but rows 8000 times smaller than the largest would lose 11 % of their y.)
#define F16_AS_IS 3
template <int DT> struct FfElem : ElemOf<DT> { static constexpr bool F16 = false; };
template <> struct FfElem<F16_AS_IS> {
    typedef _Float16 type;
    static constexpr int NP = 1;
    static constexpr bool F16 = true;
};
template <int DT> struct GateOperands { static constexpr int V = DT == ASR_T_F16 ? F16_AS_IS : DT; };
template <bool F16>
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------- operands --
// A matrix as NP planes of bf16, row-major; rows are clamped to [0, rows)
struct Planes {
    const __bf16 *p;
    int64_t ld, ps;                      // row pitch, distance of the planes (elements)
    int64_t rows;
};

// exp(-|x| .. ) with the product x log2(e) carried to twice float32: relative error 1e-7 over the whole range
__device__ __forceinline__ float exp_acc(float x) {
    x = fminf(fmaxf(x, -87.f), 88.f);
    const float hi = x * 1.44269504088896340736f;
    const float lo = __builtin_fmaf(x, 1.44269504088896340736f, -hi) + x * 1.92596299112661746887e-8f;
    const float r = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(r, lo * 0.693147180559945309417f, r);
}
// FAST: for values that are rounded to 16 bits right after, exp by one base-2 exponential (relative error 2^-24 |x|)
template <bool FAST>
__device__ __forceinline__ float exp_of(float x) { return FAST ? __builtin_amdgcn_exp2f(x * 1.44269504088896340736f) : exp_acc(x); }
template <bool FAST>
__device__ __forceinline__ void act_both(int kind, float a, float &y, float &dy) {
    if (kind == GFF_SWISH) {
        const float s = __builtin_amdgcn_rcpf(1.f + exp_of<FAST>(-a));
        y = a * s;
        dy = s * (1.f + a * (1.f - s));
    } else {
        const float cdf = 0.5f * (1.f + erff(a * 0.70710678118654752440f));
        y = a * cdf;
        dy = cdf + a * exp_of<FAST>(-0.5f * a * a) * 0.39894228040143267794f;
    }
}
__device__ __forceinline__ float act_fwd(int kind, float a) {
    float y, dy;
    act_both<false>(kind, a, y, dy);
    return y;
}

// -------------------------------------------------------------------------------------------- LDS images --
// A workgroup of the products: pieces, depth of a k-tile, LDS images of it, register sets on their way, threads, the waves'
// grid WM x WN over the tile, WK such grids that share out each k-tile's steps of 16 k, and whether operands are float16
template <int NP_, int BK_, int NBUF_, int NSET_, int NT_, int WM_, int WN_, int WK_ = 1, bool F16_ = false>
struct GemmCfg {
    static constexpr bool F16 = F16_;
    static constexpr int NP = NP_, BK = BK_, NBUF = NBUF_, NSET = NSET_, NT = NT_, WM = WM_, WN = WN_, WK = WK_;
    static_assert(NT == 64 * WM * WN * WK, "threads");
};
// Images without padding; the 16-byte chunks of a row are permuted by an exclusive or with bits of the row, so that what a
// read instruction takes at a time falls on different banks: the same chunk of 16 rows (k-contiguous image [row][BK], read with
// ds_read_b128), 64 B of four rows (row-contiguous image [k][R], read with the transposing ds_read_b64).  With padding in its
// place the writes of the 64-byte rows met on the banks: 30 % of the LDS cycles of the float32 products.
template <int BK>
__device__ __forceinline__ int nt_at(int row, int chunk) {
    return row * 2 * BK + ((chunk ^ (BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3)) << 4);
}
template <int R>
__device__ __forceinline__ int tn_at(int k, int chunk) { return k * 2 * R + ((chunk ^ ((k & 3) << 2)) << 4); }

// fragment (row r0 + lane&31, k = 16 ks + 8 (lane>>5) ..+7) of a k-contiguous image; r0 a multiple of 32
template <int BK>
__device__ __forceinline__ bf16x8 frag_nt(const unsigned char *img, int r0, int ks, int lane) {
    const u32x4p v = *reinterpret_cast<const u32x4p *>(img + r0 * 2 * BK + nt_at<BK>(lane & 31, ks * 2 + (lane >> 5)));
    return __builtin_bit_cast(bf16x8, v);
}
// the same of a row-contiguous image [k][R]: two transposing reads of 4 k x 16 rows per 16 lanes
template <int R>
__device__ __forceinline__ bf16x8 frag_tn(const unsigned char *img, int r0, int ks, int lane) {
    const int q = (lane & 15) >> 2, p = lane & 3, ch = r0 / 8 + 2 * ((lane >> 4) & 1) + (p >> 1);
    const unsigned char *a = img + (16 * ks + 8 * (lane >> 5)) * 2 * R + 8 * (p & 1);
    typedef __attribute__((address_space(3))) s16x4g *lds_p;
    const s16x4g v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + tn_at<R>(q, ch)));
    const s16x4g v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + tn_at<R>(q + 4, ch)));
    const s16x8g v = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    return __builtin_bit_cast(bf16x8, v);
}

// One operand tile of R rows x BK k: per thread R * BK / (8 NT) accesses of 16 bytes a piece
template <typename C, int R>
struct NtTile {
    static constexpr int NP = C::NP, BK = C::BK, TOT = R * BK / 8, NS = (TOT + C::NT - 1) / C::NT, IMG = R * 2 * BK;
    const __bf16 *p[NS];
    int64_t ps;
    u32x4p v[C::NSET][NP][NS];
    // PAIR: row groups of 32 alternate between the two matrices (gate, up): group g holds columns n0 + 32 (g / 2) + ...
    template <bool PAIR>
    __device__ __forceinline__ void init(const Planes &m0, const Planes &m1, int64_t r0) {
        ps = m0.ps;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int f = min((int)threadIdx.x + C::NT * i, TOT - 1), row = f / (BK / 8), kc = f % (BK / 8);
            const bool second = PAIR && ((row >> 5) & 1);
            int64_t r = r0 + (PAIR ? ((row >> 6) << 5) + (row & 31) : row);
            r = r < m0.rows ? r : m0.rows - 1;
            p[i] = (second ? m1.p : m0.p) + r * m0.ld + kc * 8;
        }
    }
    template <int S>
    __device__ __forceinline__ void load_slot(int i, int64_t k0) {
#pragma unroll
        for (int q = 0; q < NP; ++q) v[S][q][i] = *reinterpret_cast<const u32x4p *>(p[i] + q * ps + k0);
    }
    template <int S>
    __device__ __forceinline__ void store_slot(int i, unsigned char *img) const {
        const int f = threadIdx.x + C::NT * i;
        if (TOT % C::NT != 0 && f >= TOT) return;
#pragma unroll
        for (int q = 0; q < NP; ++q) *reinterpret_cast<u32x4p *>(img + q * IMG + nt_at<BK>(f / (BK / 8), f % (BK / 8))) = v[S][q][i];
    }
};
// BK rows of the matrix (the product's k) x R columns; columns past ld read column 0, rows past the matrix its last row
template <typename C, int R>
struct TnTile {
    static constexpr int NP = C::NP, BK = C::BK, NS = R * BK / 8 / C::NT, IMG = BK * 2 * R;
    static_assert(NS * 8 * C::NT == R * BK, "whole accesses");
    const __bf16 *p;
    int64_t ld, ps, rows;
    int col[NS];
    u32x4p v[C::NSET][NP][NS];
    __device__ __forceinline__ void init(const Planes &m, int64_t c0) {
        p = m.p;
        ld = m.ld;
        ps = m.ps;
        rows = m.rows;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int64_t c = c0 + ((threadIdx.x + C::NT * i) % (R / 8)) * 8;
            col[i] = c < ld ? (int)c : 0;
        }
    }
    template <int S>
    __device__ __forceinline__ void load_slot(int i, int64_t k0) {
        int64_t r = k0 + (threadIdx.x + C::NT * i) / (R / 8);
        r = r < rows ? r : rows - 1;
        const __bf16 *a = p + r * ld + col[i];
#pragma unroll
        for (int q = 0; q < NP; ++q) v[S][q][i] = *reinterpret_cast<const u32x4p *>(a + q * ps);
    }
    template <int S>
    __device__ __forceinline__ void store_slot(int i, unsigned char *img) const {
        const int f = threadIdx.x + C::NT * i;
#pragma unroll
        for (int q = 0; q < NP; ++q) *reinterpret_cast<u32x4p *>(img + q * IMG + tn_at<R>(f / (R / 8), f % (R / 8))) = v[S][q][i];
    }
};
template <int S, typename T>
__device__ __forceinline__ void load_all(T &t, int64_t k0) {
#pragma unroll
    for (int i = 0; i < T::NS; ++i) t.template load_slot<S>(i, k0);
}
template <int S, typename T>
__device__ __forceinline__ void store_all(const T &t, unsigned char *img) {
#pragma unroll
    for (int i = 0; i < T::NS; ++i) t.template store_slot<S>(i, img);
}

// acc += A B over one k-tile; fa / fb (piece, tile, ks) deliver fragments.  Smallest pieces first.
template <int NP, bool F16, int KS, int TM, int TN, typename FA, typename FB>
__device__ __forceinline__ void mma_tile(f32x16 (&acc)[TM][TN], FA fa, FB fb) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        bf16x8 a[NP][TM], b[NP][TN];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
#pragma unroll
            for (int i = 0; i < TM; ++i) a[q][i] = fa(q, i, ks);
#pragma unroll
            for (int j = 0; j < TN; ++j) b[q][j] = fb(q, j, ks);
        }
#pragma unroll
        for (int s = NP - 1; s >= 0; --s)
#pragma unroll
            for (int q = s; q >= 0; --q)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = mma<F16>(a[q][i], b[s - q][j], acc[i][j]);
    }
}

// The main loop: k-tiles [kt0, kt1) of A (TA rows) times B (TB rows); leaves the LDS free to use (ends with a barrier).
// Past the end the last tile is loaded again: its reads stay in bounds and nothing uses them.
// One image: a tile's loads run under the previous tile's products.  Two images and two register sets: while a tile is
// multiplied the next one goes from its registers to the other image and the one after it is loaded, slot by slot between the
// matrix instructions, as are the fragments of the next 16 k: one barrier a tile, and nothing waits in front of it.
template <int N> struct IntC { static constexpr int value = N; };
template <typename C, int TM, int TN, typename TA, typename TB, typename FA, typename FB>
__device__ __forceinline__ void main_loop(f32x16 (&acc)[TM][TN], TA &ta, TB &tb, unsigned char *lds, int64_t kt0, int64_t kt1,
                                          FA frag_a, FB frag_b) {
    constexpr int NP = C::NP, IA = NP * TA::IMG, IB = NP * TB::IMG;
    if (kt0 >= kt1) return;
    load_all<0>(ta, kt0 * C::BK);
    load_all<0>(tb, kt0 * C::BK);
    if constexpr (C::NBUF == 1) {
        for (int64_t kt = kt0; kt < kt1; ++kt) {
            store_all<0>(ta, lds);
            store_all<0>(tb, lds + IA);
            __syncthreads();
            if (kt + 1 < kt1) {
                load_all<0>(ta, (kt + 1) * C::BK);
                load_all<0>(tb, (kt + 1) * C::BK);
            }
            mma_tile<NP, C::F16, C::BK / 16, TM, TN>(acc, [&](int q, int i, int ks) { return frag_a(lds + q * TA::IMG, i, ks); },
                                             [&](int q, int j, int ks) { return frag_b(lds + IA + q * TB::IMG, j, ks); });
            __syncthreads();
        }
    } else {
        constexpr int KS = C::BK / 16 / C::WK, NM = TM * TN, NCH = KS * NM, NF = TM + TN, NSL = TA::NS + TB::NS;
        auto k_of = [&](int64_t kt) { return (kt < kt1 ? kt : kt1 - 1) * C::BK; };
        auto body = [&](auto tag, int64_t kt) {
            constexpr int P = decltype(tag)::value;
            const unsigned char *img = lds + P * (IA + IB);
            unsigned char *nxt = lds + (P ^ 1) * (IA + IB);
            const int64_t k2 = k_of(kt + 2);
            // (several pieces: the fragments of 16 k already fill the registers, and last for three to six times the products)
            constexpr int NFB = NP == 1 ? 2 : 1;
            bf16x8 a[NFB][NP][TM], b[NFB][NP][TN];
            auto frag = [&](int s, int ks, int f) {
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    if (f < TM) a[s][q][f] = frag_a(img + q * TA::IMG, f, ks);
                    else b[s][q][f - TM] = frag_b(img + IA + q * TB::IMG, f - TM, ks);
                }
            };
#pragma unroll
            for (int f = 0; f < NF; ++f) frag(0, 0, f);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ks = c / NM, m = c % NM, i = m / TN, j = m % TN;
                if (NFB == 2 && ks + 1 < KS) {
#pragma unroll
                    for (int f = m * NF / NM; f < (m + 1) * NF / NM; ++f) frag((ks + 1) & 1, ks + 1, f);
                }
                if (NFB == 1 && ks > 0 && m == 0) {
#pragma unroll
                    for (int f = 0; f < NF; ++f) frag(0, ks, f);
                }
#pragma unroll
                for (int s = NP - 1; s >= 0; --s)
#pragma unroll
                    for (int q = s; q >= 0; --q)
                        acc[i][j] = mma<C::F16>(a[ks % NFB][q][i], b[ks % NFB][s - q][j], acc[i][j]);
#pragma unroll
                for (int sl = c * NSL / NCH; sl < (c + 1) * NSL / NCH; ++sl) {
                    if (sl < TA::NS) {
                        ta.template store_slot<P ^ 1>(sl, nxt);
                        ta.template load_slot<P>(sl, k2);
                    } else {
                        tb.template store_slot<P ^ 1>(sl - TA::NS, nxt + IA);
                        tb.template load_slot<P>(sl - TA::NS, k2);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __syncthreads();
        };
        load_all<1>(ta, k_of(kt0 + 1));
        load_all<1>(tb, k_of(kt0 + 1));
        store_all<0>(ta, lds);
        store_all<0>(tb, lds + IA);
        __syncthreads();
        for (int64_t kt = kt0; kt < kt1; kt += 2) {
            body(IntC<0>{}, kt);
            if (kt + 1 < kt1) body(IntC<1>{}, kt + 1);
        }
    }
}

template <int TM, int TN>
__device__ __forceinline__ void zero_acc(f32x16 (&acc)[TM][TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
}

// A 32 x 32 accumulator tile (lane = column, registers = rows) turned through a wave's 4 KB of LDS: put(row, col, v) gets four
// consecutive columns of a row at a time, eight rows of 128 B per step.
template <typename F>
__device__ __forceinline__ void turn_tile(const f32x16 &t, float *S, F put) {
    const int lane = threadIdx.x & 63;
    wave_sync();
#pragma unroll
    for (int r = 0; r < 16; ++r) S[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * 32 + (lane & 31)] = t[r];
    wave_sync();
#pragma unroll
    for (int p = 0; p < 4; ++p) put(p * 8 + (lane >> 3), (lane & 7) * 4, *reinterpret_cast<const float4 *>(&S[(p * 8 + (lane >> 3)) * 32 + (lane & 7) * 4]));
    wave_sync();
}

template <int NP, bool F16>
__device__ __forceinline__ void put_pieces(__bf16 *dst, int64_t ps, float4 v) {
    if constexpr (F16) {
        *reinterpret_cast<f16x4 *>(dst) = f16x4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        return;
    }
    unsigned lo[NP], hi[NP];
    split_pair<NP>(v.x, v.y, lo);
    split_pair<NP>(v.z, v.w, hi);
#pragma unroll
    for (int q = 0; q < NP; ++q) *reinterpret_cast<u32x2p *>(dst + q * ps) = u32x2p{lo[q], hi[q]};
}
template <typename E>
__device__ __forceinline__ void put_row4(E *row, int64_t col, int64_t n, bool vec, float4 v) {
    const float t[4] = {v.x, v.y, v.z, v.w};
    if (vec && col + 3 < n) {
        store_vec<E, 4>(row + col, t);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < n) row[col + e] = (E)t[e];
    }
}

// Workgroups go to the 8 XCDs round-robin by linear id: XCD x works through one contiguous run of the tiles, column
// tiles fastest, so that the tiles that share an operand's rows share an L2.
__device__ __forceinline__ void tile_of(int id, int ntiles, int ncol, int &row, int &col) {
    const int q = ntiles >> 3, r = ntiles & 7, x = id & 7, loc = id >> 3;
    const int t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + loc;
    row = t / ncol;
    col = t - row * ncol;
}

// ------------------------------------------------------------------- a, b (and dh) of one tile, elementwise part --
struct GateParams {
    Planes x, wg, wu;                    // x (M, dp), weights (f, dp)
    Planes dy, wdt;                      // backward: dy (M, np), Wd^T (f, np)
    __bf16 *h, *dab;                     // (Mp, fp) and (Mp, 2 fp) in pieces
    int64_t h_ps, dab_ps;
    int64_t M, Mp, fp;
    int f, dp, np, ncol, ntiles, act;
};

// BM rows x BN columns of h, in OP pieces: A tile of BM rows, B tile of 2 BN (gate and up rows interleaved), then of BN rows of Wd^T
template <typename C, int OP, int BM, int BN, bool BWD>
__global__ __launch_bounds__(C::NT, 2) void gff_gate_kernel(GateParams p) {
    constexpr int NP = C::NP, TM = BM / C::WM / 32, RM = BM / C::WM;
    static_assert(BN / C::WN == 32, "a wave has the gate and the up values of 32 columns");
    typedef NtTile<C, BM> TA;
    typedef NtTile<C, 2 * BN> TB;
    typedef NtTile<C, BN> TD;
    constexpr int POOL = C::NBUF * NP * (TA::IMG + TB::IMG), TURN = C::NT / 64 * 4096;
    __shared__ __attribute__((aligned(16))) unsigned char pool[POOL > TURN ? POOL : TURN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / C::WN, wn = wave % C::WN;
    int tm, tn;
    tile_of(blockIdx.x, p.ntiles, p.ncol, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    f32x16 ab[TM][2];
    zero_acc(ab);
    {
        TA ta;
        TB tb;
        ta.template init<false>(p.x, p.x, m0);
        tb.template init<true>(p.wg, p.wu, n0);
        main_loop<C>(ab, ta, tb, pool, 0, p.dp / C::BK,
                     [&](const unsigned char *img, int i, int ks) { return frag_nt<C::BK>(img, wm * RM + i * 32, ks, lane); },
                     [&](const unsigned char *img, int j, int ks) { return frag_nt<C::BK>(img, wn * 64 + j * 32, ks, lane); });
    }
    f32x16 dh[TM][1];
    if (BWD) {
        zero_acc(dh);
        TA ta;
        TD tb;
        ta.template init<false>(p.dy, p.dy, m0);
        tb.template init<false>(p.wdt, p.wdt, n0);
        main_loop<C>(dh, ta, tb, pool, 0, p.np / C::BK,
                     [&](const unsigned char *img, int i, int ks) { return frag_nt<C::BK>(img, wm * RM + i * 32, ks, lane); },
                     [&](const unsigned char *img, int j, int ks) { return frag_nt<C::BK>(img, wn * 32 + j * 32, ks, lane); });
    }
    float *S = reinterpret_cast<float *>(pool) + wave * 1024;
    const int64_t cb = n0 + wn * 32;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t rb = m0 + wm * RM + i * 32;
        if (rb >= p.Mp) break;                                                     // a tile may reach past the padded rows
        f32x16 hh, da, db;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float y, dy;
            act_both<OP == 1>(p.act, ab[i][0][r], y, dy);
            hh[r] = y * ab[i][1][r];
            if (BWD) {
                da[r] = dh[i][0][r] * ab[i][1][r] * dy;
                db[r] = dh[i][0][r] * y;
            }
        }
        if (cb + 32 > p.f || rb + 32 > p.M) {                                      // what lies past the matrix is stored as zeros
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool ok = cb + (lane & 31) < p.f && rb + ((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) < p.M;
                hh[r] = ok ? hh[r] : 0.f;
                if (BWD) {
                    da[r] = ok ? da[r] : 0.f;
                    db[r] = ok ? db[r] : 0.f;
                }
            }
        }
        __bf16 *h = p.h + rb * p.fp + cb, *d = BWD ? p.dab + rb * 2 * p.fp + cb : nullptr;
        const int fp = (int)p.fp;
        turn_tile(hh, S, [&](int r, int c, float4 v) { put_pieces<OP, false>(h + (r * fp + c), p.h_ps, v); });
        if (BWD) {
            turn_tile(da, S, [&](int r, int c, float4 v) { put_pieces<OP, false>(d + (r * 2 * fp + c), p.dab_ps, v); });
            turn_tile(db, S, [&](int r, int c, float4 v) { put_pieces<OP, false>(d + (r * 2 * fp + fp + c), p.dab_ps, v); });
        }
    }
}

// ------------------------------------------------------------------------------------ C = A B^T, one output --
struct NtParams {
    Planes a, b;
    void *c;
    int64_t ldc, M, N, K;
    int ncol, ntiles, vec;
};
template <int DT, typename C, int BM, int BN>
__global__ __launch_bounds__(C::NT, 2) void gff_nt_kernel(NtParams p) {
    constexpr int NP = C::NP, RM = BM / C::WM, RN = BN / C::WN, TM = RM / 32, TN = RN / 32, GRID = C::WM * C::WN;
    typedef typename FfElem<DT>::type E;
    typedef NtTile<C, BM> TA;
    typedef NtTile<C, BN> TB;
    constexpr int POOL = C::NBUF * NP * (TA::IMG + TB::IMG), TURN = GRID * (4096 + (C::WK - 1) * TM * TN * 4096);
    __shared__ __attribute__((aligned(16))) unsigned char pool[POOL > TURN ? POOL : TURN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wk = wave / GRID, wm = wave % GRID / C::WN, wn = wave % C::WN;
    int tm, tn;
    tile_of(blockIdx.x, p.ntiles, p.ncol, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    f32x16 acc[TM][TN];
    zero_acc(acc);
    TA ta;
    TB tb;
    ta.template init<false>(p.a, p.a, m0);
    tb.template init<false>(p.b, p.b, n0);
    main_loop<C>(acc, ta, tb, pool, 0, p.K / C::BK,
                 [&](const unsigned char *img, int i, int ks) { return frag_nt<C::BK>(img, wm * RM + i * 32, ks * C::WK + wk, lane); },
                 [&](const unsigned char *img, int j, int ks) { return frag_nt<C::BK>(img, wn * RN + j * 32, ks * C::WK + wk, lane); });
    float *S = reinterpret_cast<float *>(pool) + wave % GRID * 1024;
    if constexpr (C::WK == 2) {                                                    // the second grid's sums join the first's
        float *J = reinterpret_cast<float *>(pool) + GRID * 1024 + wave % GRID * TM * TN * 1024;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (wk == 1) J[((i * TN + j) * 16 + r) * 64 + lane] = acc[i][j][r];
        __syncthreads();
        if (wk == 1) return;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] += J[((i * TN + j) * 16 + r) * 64 + lane];
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int64_t rb = m0 + wm * RM + i * 32, cb = n0 + wn * RN + j * 32;
            turn_tile(acc[i][j], S, [&](int r, int c, float4 v) {
                if (rb + r < p.M) put_row4<E>((E *)p.c + (rb + r) * p.ldc, cb + c, p.N, p.vec, v);
            });
        }
}

// ------------------------------------------------------------- C = A^T B over the rows, split over workgroups --
// Output row r < half goes to c0, r >= half to c1 (the gate's and the up projection's gradients lie half apart in [da db]);
// rows from `valid` on of either are padding.  With splits > 1 every split writes float32 partials, gff_sum_kernel adds them in
// order.  Both kernels take up to two products: the first one's workgroups come first.
struct TnParams {
    Planes a, b;
    void *c0, *c1;
    float *part;
    int64_t rows, half, valid, N, part_sz;
    int64_t kt, kt_split;
    int ncol, ntiles, splits, vec;
};
struct TnPair { TnParams p[2]; int blk; };
template <int DT, typename C, int BM, int BN>
__global__ __launch_bounds__(C::NT, 2) void gff_tn_kernel(TnPair pair) {
    const TnParams &p = pair.p[(int)blockIdx.x >= pair.blk];
    const int id = (int)blockIdx.x - ((int)blockIdx.x >= pair.blk ? pair.blk : 0), split = id / p.ntiles;
    constexpr int NP = C::NP, RM = BM / C::WM, RN = BN / C::WN, TM = RM / 32, TN = RN / 32;
    typedef typename FfElem<DT>::type E;
    typedef TnTile<C, BM> TA;
    typedef TnTile<C, BN> TB;
    constexpr int POOL = C::NBUF * NP * (TA::IMG + TB::IMG), TURN = C::NT / 64 * 4096;
    __shared__ __attribute__((aligned(16))) unsigned char pool[POOL > TURN ? POOL : TURN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / C::WN, wn = wave % C::WN;
    int tm, tn;
    tile_of(id - split * p.ntiles, p.ntiles, p.ncol, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    f32x16 acc[TM][TN];
    zero_acc(acc);
    TA ta;
    TB tb;
    ta.init(p.a, m0);
    tb.init(p.b, n0);
    const int64_t k0 = split * p.kt_split;
    main_loop<C>(acc, ta, tb, pool, k0, min(p.kt, k0 + p.kt_split),
                 [&](const unsigned char *img, int i, int ks) { return frag_tn<BM>(img, wm * RM + i * 32, ks, lane); },
                 [&](const unsigned char *img, int j, int ks) { return frag_tn<BN>(img, wn * RN + j * 32, ks, lane); });
    float *S = reinterpret_cast<float *>(pool) + wave * 1024;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int64_t rb = m0 + wm * RM + i * 32, cb = n0 + wn * RN + j * 32;
            turn_tile(acc[i][j], S, [&](int r, int c, float4 v) {
                int64_t row = rb + r;
                const bool second = row >= p.half;
                row -= second ? p.half : 0;
                if (row >= p.valid || (second && p.c1 == nullptr)) return;
                if (p.part) {
                    float *dst = p.part + split * p.part_sz + ((second ? p.valid : 0) + row) * p.N;
                    put_row4<float>(dst, cb + c, p.N, p.vec, v);
                } else {
                    put_row4<E>((E *)(second ? p.c1 : p.c0) + row * p.N, cb + c, p.N, p.vec, v);
                }
            });
        }
}
template <int DT, int V>
__global__ __launch_bounds__(256) void gff_sum_kernel(TnPair pair) {
    typedef typename FfElem<DT>::type E;
    const bool second = (int)blockIdx.x >= pair.blk;
    const TnParams &p = pair.p[second];
    const int64_t n0 = p.valid * p.N, nblk = second ? (int)gridDim.x - pair.blk : min((int)gridDim.x, pair.blk), blk = (int)blockIdx.x - (second ? pair.blk : 0);
    for (int64_t i = (blk * 256 + threadIdx.x) * V; i < p.part_sz; i += nblk * 256 * V) {
        float v[V], t[V];
        load_vec<float, V>(p.part + i, v);
        for (int s = 1; s < p.splits; ++s) {
            load_vec<float, V>(p.part + s * p.part_sz + i, t);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += t[e];
        }
        store_vec<E, V>(i < n0 ? (E *)p.c0 + i : (E *)p.c1 + (i - n0), v);
    }
}

// ---------------------------------------------------------------------------------------- packing into planes --
// Up to 9 matrices in one launch: src (R, C) row-major with pitch lds -> pieces, straight (R, >= C, pitch ldd) or transposed
// (C, >= R); columns of the result from the matrix' end to `wide` are zeros.
struct PackJob {
    const void *src;
    __bf16 *dst;
    int64_t lds, ldd, ps;
    int R, C, wide, trans, vec, as_is;   // as_is: float16 as it lies instead of as pieces
    int blk0;                            // first workgroup of the job
    int nx;                              // workgroups along the source's columns
};
struct PackJobs { PackJob j[9]; int n; };

template <int DT>
__global__ __launch_bounds__(256) void gff_pack_kernel(PackJobs jobs) {
    typedef typename FfElem<DT>::type E;
    constexpr int NP = FfElem<DT>::NP;
    __shared__ float tile[64][65];
    int k = 0;
    while (k + 1 < jobs.n && (int)blockIdx.x >= jobs.j[k + 1].blk0) ++k;
    const PackJob &J = jobs.j[k];
    auto put = [&](__bf16 *dst, float4 v) {
        if (DT == ASR_T_F16 && J.as_is) put_pieces<1, true>(dst, 0, v);
        else put_pieces<NP, false>(dst, J.ps, v);
    };
    const int b = (int)blockIdx.x - J.blk0, by = b / J.nx, bx = b - by * J.nx;
    const E *src = (const E *)J.src;
    // a 64 x 64 block; source columns (or, transposed, rows) past the end read as zero.  All loads of a thread go out together.
    const int tc = (threadIdx.x & 15) * 4, tr = threadIdx.x >> 4, r0 = by * 64 + tr, c0 = bx * 64 + tc;
    float v[4][4];
    if (J.vec != 0 && by * 64 + 64 <= J.R && bx * 64 + 64 <= J.C) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_vec<E, 4>(src + (int64_t)(r0 + 16 * i) * J.lds + c0, v[i]);
    } else {
        E t[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) t[i][e] = src[(int64_t)min(r0 + 16 * i, J.R - 1) * J.lds + min(c0 + e, J.C - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = r0 + 16 * i < J.R && c0 + e < J.C ? (float)t[i][e] : 0.f;
    }
    if (J.trans == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (r0 + 16 * i < J.R && c0 < J.wide)
                put(J.dst + (int64_t)(r0 + 16 * i) * J.ldd + c0, make_float4(v[i][0], v[i][1], v[i][2], v[i][3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[tr + 16 * i][tc + e] = v[i][e];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = bx * 64 + tr + 16 * i, r = by * 64 + tc;                 // row and column of the result
        if (c < J.C && r < J.wide)
            put(J.dst + (int64_t)c * J.ldd + r,
                make_float4(tile[tc][tr + 16 * i], tile[tc + 1][tr + 16 * i], tile[tc + 2][tr + 16 * i], tile[tc + 3][tr + 16 * i]));
    }
}

// ------------------------------------------------------------------------------------------- a few rows: tokens --
// M <= 64 rows, forward only: the weights are read once from memory, which bounds it.  16 weight rows a workgroup, its waves
// (and, for the second product, `splits` workgroups) share k, rows of x in groups of 16; the loads of four steps of 32 k are
// in flight.  16-bit weights are multiplied as their bf16 pieces (v_mfma_f32_16x16x32_bf16), the hidden values, which stay
// float32 in between, as two; float32 weights exactly in v_mfma_f32_16x16x4_f32.  GATE: two weight matrices and h =
// act(a) b to float32 h.  Otherwise y, or, with several workgroups a tile, float32 parts that gff_few_join_kernel adds in their
// order (a last-arriver sum in the same launch took 65 us more: its device-wide fences write back the L2s).
template <int DT> struct FewPieces { static constexpr int W = DT == ASR_T_BF16 ? 1 : 2; };
template <int P>
__device__ __forceinline__ void few_split(const float (&v)[8], bf16x8 (&o)[P]) {
    u32x4p w[P];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned x[P];
        split_pair<P>(v[2 * e], v[2 * e + 1], x);
#pragma unroll
        for (int q = 0; q < P; ++q) w[q][e] = x[q];
    }
#pragma unroll
    for (int q = 0; q < P; ++q) o[q] = __builtin_bit_cast(bf16x8, w[q]);
}
template <int DT, int NM, int NW, bool GATE>
__device__ __forceinline__ void few_rows_body(const typename ElemOf<DT>::type *wa, const typename ElemOf<DT>::type *wb,
                                              const void *xin, bool vec, int64_t K, int64_t kb, int64_t ke, int M, int64_t N, int act,
                                              float *h, typename ElemOf<DT>::type *y, float *part, float *red) {
    typedef typename ElemOf<DT>::type E;
    constexpr int V = 8, NS = GATE ? 2 : 1, NA = NS * NM;            // k per lane and step: 32 k of a row over its four lanes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int64_t n = (int64_t)blockIdx.x * 16 + c, row = n < N ? n : N - 1;
    f32x4 acc[NS][NM];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[s][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const E *rw[2] = {wa + row * K, GATE ? wb + row * K : wa};
    auto fetch = [&](const auto *a, int64_t k, float (&v)[V]) {      // eight of a row, zeros past the end
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = 0.f;
        if (vec) {                                                   // K % 8 == 0: a lane's eight are all there or none is
            if (k < ke) load_vec<std::remove_const_t<std::remove_pointer_t<decltype(a)>>, V>(a + k, v);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (k + e < ke) v[e] = (float)a[k + e];
        }
    };
#pragma unroll 4
    for (int64_t k0 = kb + (int64_t)wave * 32; k0 < ke; k0 += NW * 32) {
        const int64_t k = k0 + g * V;
        float vw[NS][V], vx[NM][V];
#pragma unroll
        for (int s = 0; s < NS; ++s) fetch(rw[s], k, vw[s]);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            const int64_t r = min(m * 16 + c, M - 1);
            if constexpr (GATE) fetch((const E *)xin + r * K, k, vx[m]);
            else fetch((const float *)xin + r * K, k, vx[m]);
        }
        if constexpr (DT == ASR_T_F32) {
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int s = 0; s < NS; ++s) acc[s][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(vw[s][e], vx[m][e], acc[s][m], 0, 0, 0);
        } else {
            constexpr int PW = FewPieces<DT>::W, PX = GATE ? PW : 2, TOP = (PW > PX ? PW : PX) - 1;
            bf16x8 w[NS][PW], x[PX];
#pragma unroll
            for (int s = 0; s < NS; ++s) few_split<PW>(vw[s], w[s]);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                few_split<PX>(vx[m], x);
#pragma unroll
                for (int u = TOP; u >= 0; --u)
#pragma unroll
                    for (int q = 0; q < PW; ++q)
#pragma unroll
                        for (int s = 0; s < NS; ++s)
                            if (u - q >= 0 && u - q < PX) acc[s][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[s][q], x[u - q], acc[s][m], 0, 0, 0);
            }
        }
    }
    // D: column = x row (lane & 15), rows 4 g + r = weight rows; partials of the waves through LDS
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int m = 0; m < NM; ++m) *reinterpret_cast<f32x4 *>(red + ((wave * NA + s * NM + m) * 64 + lane) * 4) = acc[s][m];
    __syncthreads();
    const int t = threadIdx.x, m = t >> 6, l = t & 63, r = m * 16 + (l & 15);
    if (t >= NM * 64) return;
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        a += *reinterpret_cast<const f32x4 *>(red + ((w * NA + m) * 64 + l) * 4);
        if (GATE) b += *reinterpret_cast<const f32x4 *>(red + ((w * NA + NM + m) * 64 + l) * 4);
    }
    if (r >= M) return;
    const int64_t o = (int64_t)blockIdx.x * 16 + (l >> 4) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (o + e >= N) continue;
        if (GATE) h[r * N + o + e] = act_fwd(act, a[e]) * b[e];
        else if (gridDim.y > 1) part[((int64_t)blockIdx.y * M + r) * N + o + e] = a[e];
        else y[r * N + o + e] = (E)a[e];
    }
}
#define FEW_NW 8
template <int DT, int NM>
__global__ __launch_bounds__(64 * FEW_NW) void gff_few_gate_kernel(const void *x, const void *wg, const void *wu, float *h, int64_t d,
                                                                   int64_t f, int M, int act, int vec) {
    __shared__ __attribute__((aligned(16))) float red[FEW_NW * 2 * NM * 256];
    typedef typename ElemOf<DT>::type E;
    few_rows_body<DT, NM, FEW_NW, true>((const E *)wg, (const E *)wu, x, vec, d, 0, d, M, f, act, h, nullptr, nullptr, red);
}
template <int DT, int NM>
__global__ __launch_bounds__(64 * FEW_NW) void gff_few_down_kernel(const float *h, const void *wd, void *y, int64_t f, int64_t n, int M,
                                                                   int vec, int64_t run, float *part) {
    __shared__ __attribute__((aligned(16))) float red[FEW_NW * NM * 256];
    typedef typename ElemOf<DT>::type E;
    const int64_t kb = min(f, (int64_t)blockIdx.y * run), ke = min(f, kb + run);
    few_rows_body<DT, NM, FEW_NW, false>((const E *)wd, nullptr, h, vec, f, kb, ke, M, n, 0, nullptr, (E *)y, part, red);
}
template <int DT>
__global__ __launch_bounds__(256) void gff_few_join_kernel(const float *__restrict__ part, void *y, int64_t sz, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= sz) return;
    float a = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) a += part[s * sz + i];
    ((typename ElemOf<DT>::type *)y)[i] = (typename ElemOf<DT>::type)a;
}

// ------------------------------------------------------------------------------------------------------- host --
static int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// A weight gradient (rows x cols, summed over M): the tile, and in how many runs of M it is summed.  A run has at least 8
// k-tiles, and there are runs until the launch has two workgroups of four waves (or one of eight) for each compute unit.
// Where both gradients take the small tile they share their launches, which then neither fills the GPU alone (1003 x 200 x 683
// float16: 14 + 14 us for the products and 4 + 4 for their sums become 17 and 4).
struct TnPlan { int big, splits; };
static TnPlan gff_tn_plan(int NP, int64_t rows, int64_t cols, int64_t M) {
    const int64_t kt = cdiv(M, NP == 1 ? 64 : 32);
    auto runs = [&](int64_t tiles, int64_t want) {
        int64_t s = want / (tiles > 0 ? tiles : 1);
        if (s > kt / 8) s = kt / 8;
        if (s > 32) s = 32;
        return s < 1 ? 1 : (int)s;
    };
    const int64_t mid = (int64_t)cdiv(rows, 256) * cdiv(cols, 128), small = (int64_t)cdiv(rows, 128) * cdiv(cols, 128);
    const int sm = runs(mid, 256);
    if (mid * sm >= 192) return TnPlan{1, sm};
    return TnPlan{0, runs(small, 512)};
}

struct GffPlan {
    int NP, NG;                          // pieces of h, da, db and what they are multiplied by; of the gate kernel's operands
    int64_t dp, np, fp, Mp;              // padded widths of x / dy / h and rows of h, [da db]
    bool direct_x, direct_wgu, direct_wd, direct_dy;
    TnPlan gu, wd;                       // the weight gradients of [gate; up] and down
    int64_t off[16], bytes;              // workspace: byte offsets
};
enum { O_X, O_WG, O_WU, O_WD, O_H, O_DY, O_WDT, O_WGUT, O_DAB, O_PART, O_PART_WD, O_XP, O_DYP };

static bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }

// A 16-bit matrix whose k is whole k-tiles is an operand as it lies; every other one is packed into the workspace, float16 x and
// dy once for the gate kernel and once, as pieces, for the weight gradients.
static void gff_plan(const asr_gated_ff_args *a, bool bwd, GffPlan &p) {
    p.NP = a->dtype == ASR_T_F32 ? 3 : a->dtype == ASR_T_F16 ? 2 : 1;
    p.NG = a->dtype == ASR_T_F32 ? 3 : 1;
    p.dp = up_to(a->d, 64);
    p.np = up_to(a->n, 64);
    p.fp = up_to(a->f, 64);
    p.Mp = up_to(a->M, 128);
    const bool one = p.NG == 1;
    p.direct_x = one && p.dp == a->d && aligned16(a->x);
    p.direct_wgu = one && p.dp == a->d && aligned16(a->wg) && aligned16(a->wu);
    p.direct_wd = p.NP == 1 && p.fp == a->f && aligned16(a->wd);
    p.direct_dy = one && p.np == a->n && aligned16(a->dy);
    int64_t o = 0;
    auto take = [&](int k, int64_t bytes) {
        p.off[k] = o;
        o += up_to(bytes, 256);
    };
    const int64_t e = 2 * p.NP, eg = 2 * p.NG;
    take(O_X, p.direct_x ? 0 : a->M * p.dp * eg);
    take(O_WG, p.direct_wgu ? 0 : (int64_t)a->f * p.dp * eg);
    take(O_WU, p.direct_wgu ? 0 : (int64_t)a->f * p.dp * eg);
    take(O_H, p.Mp * p.fp * e);
    take(O_WD, p.direct_wd || bwd ? 0 : (int64_t)a->n * p.fp * e);
    if (bwd) {
        take(O_DY, p.direct_dy ? 0 : a->M * p.np * eg);
        take(O_WDT, (int64_t)a->f * p.np * eg);
        take(O_WGUT, (int64_t)a->d * 2 * p.fp * e);
        take(O_DAB, p.Mp * 2 * p.fp * e);
        take(O_XP, p.NP == p.NG ? 0 : a->M * p.dp * e);
        take(O_DYP, p.NP == p.NG ? 0 : a->M * p.np * e);
        p.gu = gff_tn_plan(p.NP, 2 * p.fp, a->d, a->M);
        p.wd = gff_tn_plan(p.NP, a->n, a->f, a->M);
        take(O_PART, p.gu.splits > 1 ? (int64_t)p.gu.splits * 2 * a->f * a->d * 4 : 0);
        take(O_PART_WD, p.wd.splits > 1 ? (int64_t)p.wd.splits * a->n * a->f * 4 : 0);
    }
    p.bytes = o;
}

#define GFF_FEW_ROWS 64
static bool gff_few(const asr_gated_ff_args *a) { return a->M <= GFF_FEW_ROWS; }
// The second product's workgroups: two for each compute unit, each with at least 256 k
struct FewPlan { int64_t h, part, bytes, run; int splits, tiles; };
static FewPlan gff_few_plan(const asr_gated_ff_args *a) {
    FewPlan p;
    p.tiles = cdiv(a->n, 16);
    int64_t s = 512 / p.tiles;
    if (s > a->f / 256) s = a->f / 256;
    if (s < 1) s = 1;
    p.run = up_to((a->f + s - 1) / s, 32);
    p.splits = cdiv(a->f, p.run);
    p.h = 0;
    p.part = up_to((int64_t)a->M * a->f * 4, 256);
    p.bytes = p.part + (p.splits > 1 ? (int64_t)p.splits * a->M * a->n * 4 : 0);
    return p;
}

static int gff_check(const asr_gated_ff_args *a, const char *who, bool ptrs) {
    ASR_CHECK_ARG(a, "%s: null pointer", who);
    ASR_CHECK_ARG(a->dtype >= 0 && a->dtype <= 2, "%s: unknown element type", who);
    ASR_CHECK_ARG(a->act == GFF_SWISH || a->act == GFF_GELU, "%s: unknown activation", who);
    ASR_CHECK_ARG(a->M > 0 && a->d > 0 && a->f > 0 && a->n > 0, "%s: empty shape", who);
    ASR_CHECK_ARG(a->d <= (1 << 20) && a->f <= (1 << 20) && a->n <= (1 << 20), "%s: widths are at most 2^20", who);
    ASR_CHECK_ARG((int64_t)cdiv(a->M, 128) * cdiv(a->f > a->d ? (a->f > a->n ? a->f : a->n) : (a->d > a->n ? a->d : a->n), 64) < (1ll << 30),
                  "%s: too many rows", who);
    ASR_CHECK_ARG(a->M <= (1ll << 30), "%s: at most 2^30 rows", who);
    if (ptrs) ASR_CHECK_ARG(a->x && a->wg && a->wu && a->wd && a->ws, "%s: null pointer", who);
    return ASR_OK;
}

extern "C" int64_t asr_gated_ff_ws_bytes(const asr_gated_ff_args *a, int backward) {
    if (gff_check(a, "gated_ff_ws_bytes", false) != ASR_OK) return -1;
    if (!backward && gff_few(a)) return gff_few_plan(a).bytes;
    GffPlan p;
    gff_plan(a, backward != 0, p);
    return p.bytes;
}

static void pack_add(PackJobs &j, int64_t &blocks, const void *src, void *dst, int64_t R, int64_t C, int64_t ldd, int64_t ps, int64_t wide, int trans, bool as_is) {
    PackJob &k = j.j[j.n++];
    k.src = src;
    k.dst = (__bf16 *)dst;
    k.lds = C;
    k.ldd = ldd;
    k.ps = ps;
    k.R = (int)R;
    k.C = (int)C;
    k.wide = (int)wide;
    k.trans = trans;
    k.as_is = as_is;
    k.vec = C % 4 == 0 && (uintptr_t)src % 16 == 0;
    k.blk0 = (int)blocks;
    // straight: the padding columns belong to the last blocks of a row; transposed: to the last blocks of a column
    k.nx = cdiv(trans ? C : wide, 64);
    blocks += (int64_t)k.nx * cdiv(trans ? wide : R, 64);
}

// Workgroups of the products.  One piece: eight waves, 256 x 256 or 256 x 128 (a wave's 128 x 64 or 64 x 64): with four waves
// and 128 x 128 the LDS was the bound, its writes and reads as long as the matrix work (8192 x 1024 x 4096 bfloat16: 133 us
// a product, 75 without loads and LDS writes).  Several pieces: three to six products an LDS byte, 128 x 128 with four waves.
// Smaller tiles where larger ones would leave compute units without one.
template <int DT> struct Cfg {
    static constexpr int NP = FfElem<DT>::NP, BK = NP == 1 ? 64 : 32;
    static constexpr bool F16 = FfElem<DT>::F16;
    typedef GemmCfg<1, 64, 2, 2, 512, 2, 4, 1, F16> Big;                            // 256 x 256, one piece
    typedef GemmCfg<1, 32, 2, 2, 512, 2, 4, 1, F16> Gate;                           // gate tiles of 256 x 128, one piece
    typedef GemmCfg<NP, BK, 2, 2, 512, 4, 2, 1, F16> Mid;                           // 256 x 128
    typedef GemmCfg<NP, BK, 2, 2, 512, 1, 4, 2, F16> Half;                          // 96 x 128, two grids of waves
    typedef GemmCfg<NP, BK, NP == 1 ? 2 : 1, NP == 1 ? 2 : 1, 256, 2, 2, 1, F16> Small;
    typedef GemmCfg<NP, BK, 2, 2, 256, 2, 2, 1, F16> Deep;
};

template <int DT, typename C, int BM, int BN>
static int gff_nt_go(NtParams &p, hipStream_t st) {
    p.ncol = cdiv(p.N, BN);
    p.ntiles = cdiv(p.M, BM) * p.ncol;
    hipLaunchKernelGGL((gff_nt_kernel<DT, C, BM, BN>), dim3(p.ntiles), dim3(C::NT), 0, st, p);
    ASR_CHECK_LAUNCH("gff_nt_kernel");
    return ASR_OK;
}
template <int DT>
static int gff_nt(const Planes &a, const Planes &b, void *c, int64_t M, int64_t N, int64_t K, hipStream_t st) {
    constexpr int NP = FfElem<DT>::NP;
    NtParams p{a, b, c, N, M, N, K, 0, 0, (int)(N % 4 == 0 && aligned16(c))};
    // The tile that is done first: the compute unit with most tiles has ceil(tiles / 256) of them; `rate` is the matrix work a
    // unit does in a time, `one` the share of it that a lone workgroup reaches where two or three are meant to share the unit
    // (from float32 products of 11968 x 256, k 2048 and 4096, bfloat16 ones of 8192 x 1024: 256 x 128 reaches 1.4 PFLOP/s
    // scaled to all units, 128 x 64 two a unit 0.9)
    auto time = [&](int bm, int bn, double rate, double one) {
        const int64_t n = ((int64_t)cdiv(M, bm) * cdiv(N, bn) + 255) / 256;
        return (double)n * bm * bn / (n == 1 ? rate * one : rate);
    };
    const double t256 = NP == 1 ? time(256, 256, 1.0, 1.0) : 1e300, tmid = time(256, 128, 0.95, 1.0), t96 = time(96, 128, 0.85, 1.0),
                 t128 = time(128, 64, 0.6, 0.7), t64 = time(64, 64, 0.55, 0.9);
    const double best = fmin(fmin(fmin(t256, tmid), fmin(t96, t128)), t64);
    if constexpr (NP == 1)
        if (t256 == best) return gff_nt_go<DT, typename Cfg<DT>::Big, 256, 256>(p, st);
    if (tmid == best) return gff_nt_go<DT, typename Cfg<DT>::Mid, 256, 128>(p, st);
    if (t96 == best) return gff_nt_go<DT, typename Cfg<DT>::Half, 96, 128>(p, st);
    if (t128 == best) return gff_nt_go<DT, typename Cfg<DT>::Deep, 128, 64>(p, st);
    return gff_nt_go<DT, typename Cfg<DT>::Deep, 64, 64>(p, st);
}

template <typename C, int OP, int BM, int BN, bool BWD>
static int gff_gate_go(GateParams &g, hipStream_t st) {
    g.ncol = cdiv(g.fp, BN);
    g.ntiles = cdiv(g.Mp, BM) * g.ncol;
    hipLaunchKernelGGL((gff_gate_kernel<C, OP, BM, BN, BWD>), dim3(g.ntiles), dim3(C::NT), 0, st, g);
    ASR_CHECK_LAUNCH("gff_gate_kernel");
    return ASR_OK;
}
template <int DT, bool BWD>
static int gff_gate(GateParams &g, hipStream_t st) {
    typedef Cfg<GateOperands<DT>::V> G;
    constexpr int NP = G::NP, OP = FfElem<DT>::NP;
    const int64_t rows = cdiv(g.Mp, 256);
    if constexpr (NP == 1) {
        // One piece is bound by the LDS: a wave's 128 x 32 of each product reads 16 B per matrix instruction less than 64 x 32
        // (8192 x 1024 x 4096: 298 -> 274 us with dh, 170 -> 163 us without; k-tiles of 64 would spill, 351 us).  A unit's
        // rounds of these tiles against those of half their size:
        const int64_t wide = (rows * (g.fp / 128) + 255) / 256, narrow = (rows * (g.fp / 64) + 255) / 256;
        if (g.fp % 128 == 0 && 1.85 * (double)wide <= (double)narrow) return gff_gate_go<typename G::Gate, OP, 256, 128, BWD>(g, st);
    }
    if (rows * (g.fp / 64) >= 256) return gff_gate_go<typename G::Mid, OP, 256, 64, BWD>(g, st);
    // (1003 x 200 x 683 float16, 88 tiles of 128 x 64: 17.4 us with dh and 13.2 without, in tiles of 64 x 64 12.2 and 9.2)
    if ((int64_t)cdiv(g.Mp, 128) * (g.fp / 64) < 256) return gff_gate_go<typename G::Deep, OP, 64, 64, BWD>(g, st);
    return gff_gate_go<typename G::Small, OP, 128, 64, BWD>(g, st);
}

template <int DT, typename C, int BM, int BN>
static void gff_tn_go(TnPair &pair, int n, int64_t M, hipStream_t st) {
    int64_t blocks = 0;
    for (int k = 0; k < n; ++k) {
        TnParams &p = pair.p[k];
        p.ncol = cdiv(p.N, BN);
        p.ntiles = cdiv(p.rows, BM) * p.ncol;
        p.kt = cdiv(M, C::BK);
        p.kt_split = (p.kt + p.splits - 1) / p.splits;
        blocks += (int64_t)p.ntiles * p.splits;
        if (k == 0) pair.blk = (int)blocks;
    }
    hipLaunchKernelGGL((gff_tn_kernel<DT, C, BM, BN>), dim3((unsigned)blocks), dim3(C::NT), 0, st, pair);
}
// n = 1 or 2 products with the same tile
template <int DT>
static int gff_tn(TnPair &pair, int n, int big, int64_t M, hipStream_t st) {
    if (big) gff_tn_go<DT, typename Cfg<DT>::Mid, 256, 128>(pair, n, M, st);
    else gff_tn_go<DT, typename Cfg<DT>::Small, 128, 128>(pair, n, M, st);
    ASR_CHECK_LAUNCH("gff_tn_kernel");
    TnPair sums{};
    int m = 0, blocks = 0;
    bool vec = true;
    for (int k = 0; k < n; ++k)
        if (pair.p[k].splits > 1) {
            const TnParams &p = sums.p[m++] = pair.p[k];
            vec = vec && p.valid * p.N % 4 == 0 && aligned16(p.c0) && aligned16(p.c1);
        }
    if (!m) return ASR_OK;
    for (int k = 0; k < m; ++k) {
        const int need = cdiv(sums.p[k].part_sz, vec ? 1024 : 256);
        blocks += need < 4096 ? need : 4096;
        if (k == 0) sums.blk = blocks;
    }
    if (vec) hipLaunchKernelGGL((gff_sum_kernel<DT, 4>), dim3(blocks), dim3(256), 0, st, sums);
    else hipLaunchKernelGGL((gff_sum_kernel<DT, 1>), dim3(blocks), dim3(256), 0, st, sums);
    ASR_CHECK_LAUNCH("gff_sum_kernel");
    return ASR_OK;
}

template <int DT>
static int gff_run(const asr_gated_ff_args *a, bool bwd, hipStream_t st) {
    constexpr bool TWICE = DT == ASR_T_F16;            // x and dy as they lie for the gate kernel and as pieces for the weight gradients
    GffPlan p;
    gff_plan(a, bwd, p);
    char *ws = (char *)a->ws;
    auto at = [&](int k) { return (__bf16 *)(ws + p.off[k]); };
    Planes x{p.direct_x ? (const __bf16 *)a->x : at(O_X), p.dp, a->M * p.dp, a->M};
    Planes wg{p.direct_wgu ? (const __bf16 *)a->wg : at(O_WG), p.dp, (int64_t)a->f * p.dp, a->f};
    Planes wu{p.direct_wgu ? (const __bf16 *)a->wu : at(O_WU), p.dp, (int64_t)a->f * p.dp, a->f};
    Planes wd{p.direct_wd ? (const __bf16 *)a->wd : at(O_WD), p.fp, (int64_t)a->n * p.fp, a->n};
    Planes h{at(O_H), p.fp, p.Mp * p.fp, p.Mp};
    Planes dy{}, wdt{}, wgut{}, dab{}, xp{}, dyp{};
    PackJobs jobs;
    jobs.n = 0;
    int64_t blocks = 0;
    if (!p.direct_x) pack_add(jobs, blocks, a->x, at(O_X), a->M, a->d, p.dp, x.ps, p.dp, 0, TWICE);
    if (!p.direct_wgu) {
        pack_add(jobs, blocks, a->wg, at(O_WG), a->f, a->d, p.dp, wg.ps, p.dp, 0, TWICE);
        pack_add(jobs, blocks, a->wu, at(O_WU), a->f, a->d, p.dp, wu.ps, p.dp, 0, TWICE);
    }
    if (!bwd && !p.direct_wd) pack_add(jobs, blocks, a->wd, at(O_WD), a->n, a->f, p.fp, wd.ps, p.fp, 0, false);
    if (bwd) {
        dy = Planes{p.direct_dy ? (const __bf16 *)a->dy : at(O_DY), p.np, a->M * p.np, a->M};
        wdt = Planes{at(O_WDT), p.np, (int64_t)a->f * p.np, a->f};
        wgut = Planes{at(O_WGUT), 2 * p.fp, (int64_t)a->d * 2 * p.fp, a->d};
        dab = Planes{at(O_DAB), 2 * p.fp, p.Mp * 2 * p.fp, p.Mp};
        xp = TWICE ? Planes{at(O_XP), p.dp, a->M * p.dp, a->M} : x;
        dyp = TWICE ? Planes{at(O_DYP), p.np, a->M * p.np, a->M} : dy;
        if (!p.direct_dy) pack_add(jobs, blocks, a->dy, at(O_DY), a->M, a->n, p.np, dy.ps, p.np, 0, TWICE);
        pack_add(jobs, blocks, a->wd, at(O_WDT), a->n, a->f, p.np, wdt.ps, p.np, 1, TWICE);
        pack_add(jobs, blocks, a->wg, at(O_WGUT), a->f, a->d, 2 * p.fp, wgut.ps, p.fp, 1, false);
        pack_add(jobs, blocks, a->wu, at(O_WGUT) + p.fp, a->f, a->d, 2 * p.fp, wgut.ps, p.fp, 1, false);
        if (TWICE && a->dwg) pack_add(jobs, blocks, a->x, at(O_XP), a->M, a->d, p.dp, xp.ps, p.dp, 0, false);
        if (TWICE && a->dwd) pack_add(jobs, blocks, a->dy, at(O_DYP), a->M, a->n, p.np, dyp.ps, p.np, 0, false);
    }
    if (jobs.n) {
        ASR_CHECK_ARG(blocks < (1ll << 31), "gated_ff: too many rows");
        hipLaunchKernelGGL((gff_pack_kernel<DT>), dim3((unsigned)blocks), dim3(256), 0, st, jobs);
        ASR_CHECK_LAUNCH("gff_pack_kernel");
    }
    GateParams g{x, wg, wu, dy, wdt, (__bf16 *)h.p, (__bf16 *)dab.p, h.ps, dab.ps, a->M, p.Mp, p.fp, a->f, (int)p.dp, (int)p.np, 0, 0, a->act};
    if (!bwd) {
        ASR_CHECK((gff_gate<DT, false>(g, st)));
        return gff_nt<DT>(h, wd, a->y, a->M, a->n, p.fp, st);
    }
    ASR_CHECK((gff_gate<DT, true>(g, st)));
    if (a->dx) ASR_CHECK(gff_nt<DT>(dab, wgut, a->dx, a->M, a->d, 2 * p.fp, st));
    const TnParams gu{dab, xp, a->dwg, a->dwu, p.gu.splits > 1 ? (float *)at(O_PART) : nullptr, 2 * p.fp, p.fp, a->f, a->d, 2ll * a->f * a->d, 0, 0, 0, 0,
                      p.gu.splits, (int)(a->d % 4 == 0 && aligned16(a->dwg) && aligned16(a->dwu))};
    const TnParams down{dyp, h, a->dwd, nullptr, p.wd.splits > 1 ? (float *)at(O_PART_WD) : nullptr, a->n, up_to(a->n, 256), a->n, a->f, (int64_t)a->n * a->f,
                        0, 0, 0, 0, p.wd.splits, (int)(a->f % 4 == 0 && aligned16(a->dwd))};
    TnPair both{{gu, down}, 0}, one{{gu}, 0}, other{{down}, 0};
    if (a->dwg && a->dwd && !p.gu.big && !p.wd.big) return gff_tn<DT>(both, 2, 0, a->M, st);
    if (a->dwg) ASR_CHECK(gff_tn<DT>(one, 1, p.gu.big, a->M, st));
    if (a->dwd) ASR_CHECK(gff_tn<DT>(other, 1, p.wd.big, a->M, st));
    return ASR_OK;
}

template <int DT, int NM>
static int gff_few_run(const asr_gated_ff_args *a, hipStream_t st) {
    const FewPlan p = gff_few_plan(a);
    char *ws = (char *)a->ws;
    float *h = (float *)(ws + p.h), *part = (float *)(ws + p.part);
    hipLaunchKernelGGL((gff_few_gate_kernel<DT, NM>), dim3(cdiv(a->f, 16)), dim3(64 * FEW_NW), 0, st, a->x, a->wg, a->wu, h, (int64_t)a->d,
                       (int64_t)a->f, (int)a->M, a->act, (int)(a->d % 8 == 0 && aligned16(a->x) && aligned16(a->wg) && aligned16(a->wu)));
    hipLaunchKernelGGL((gff_few_down_kernel<DT, NM>), dim3(p.tiles, p.splits), dim3(64 * FEW_NW), 0, st, (const float *)h, a->wd, a->y,
                       (int64_t)a->f, (int64_t)a->n, (int)a->M, (int)(a->f % 8 == 0 && aligned16(a->wd) && aligned16(a->ws)), p.run, part);
    if (p.splits > 1)
        hipLaunchKernelGGL((gff_few_join_kernel<DT>), dim3(cdiv((int64_t)a->M * a->n, 256)), dim3(256), 0, st, (const float *)part, a->y,
                           (int64_t)a->M * a->n, p.splits);
    ASR_CHECK_LAUNCH("gff_few_kernel");
    return ASR_OK;
}
template <int DT>
static int gff_few_pick(const asr_gated_ff_args *a, hipStream_t st) {
    return a->M <= 16 ? gff_few_run<DT, 1>(a, st) : a->M <= 32 ? gff_few_run<DT, 2>(a, st) : gff_few_run<DT, 4>(a, st);
}

extern "C" int asr_gated_ff_fwd(const asr_gated_ff_args *a, void *stream) {
    ASR_CHECK(gff_check(a, "gated_ff_fwd", true));
    ASR_CHECK_ARG(a->y, "gated_ff_fwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const bool few = gff_few(a);
    switch (a->dtype) {
        case ASR_T_F32: return few ? gff_few_pick<ASR_T_F32>(a, st) : gff_run<ASR_T_F32>(a, false, st);
        case ASR_T_BF16: return few ? gff_few_pick<ASR_T_BF16>(a, st) : gff_run<ASR_T_BF16>(a, false, st);
        default: return few ? gff_few_pick<ASR_T_F16>(a, st) : gff_run<ASR_T_F16>(a, false, st);
    }
}

extern "C" int asr_gated_ff_bwd(const asr_gated_ff_args *a, void *stream) {
    ASR_CHECK(gff_check(a, "gated_ff_bwd", true));
    ASR_CHECK_ARG(a->dy, "gated_ff_bwd: null pointer");
    ASR_CHECK_ARG((a->dwg == nullptr) == (a->dwu == nullptr), "gated_ff_bwd: dwg and dwu come together");
    hipStream_t st = (hipStream_t)stream;
    switch (a->dtype) {
        case ASR_T_F32: return gff_run<ASR_T_F32>(a, true, st);
        case ASR_T_BF16: return gff_run<ASR_T_BF16>(a, true, st);
        default: return gff_run<ASR_T_F16>(a, true, st);
    }
}
