// Cross attention: queries of one sequence against keys / values of another one, softmax(scale q k^T) v per head, with a key padding
// mask, shared key / value heads and the backward pass.  Included by one unit per element type (xattn_f32 / _bf16 / _f16.hip) and by the
// host side (xattn.hip).
//
// One pass over the keys with a running maximum and sum (no score matrix in memory).  Every product is a 32x32x16 16-bit MFMA:
//   * the streamed operand (K, V forward and dQ; Q, dO for dK / dV) is staged row-major in LDS; as an MFMA A operand its rows are read
//     with ds_read_b128, transposed with ds_read_b64_tr_b16 (4 rows x 16 columns per 16 lanes);
//   * the stationary operand sits in registers as B operand, so that a score tile comes out TRANSPOSED: lane l owns query (or key)
//     l % 32 and holds 16 scores of it.  Row statistics are per-lane scalars (one lane exchange per tile), and the tile's registers are,
//     packed, the B operand of the next product: contraction slot (l / 32, j) of step s is row 16 s + 8 (j / 4) + 4 (l / 32) + j % 4 of
//     the tile, and the transposed LDS read delivers the same order.  Probabilities never pass through LDS.
//   * fp32 elements are split into three bf16 planes (24 significand bits, fp32's exponent range) and multiplied with six products, the
//     dropped ones are below 2^-24 of the operands' product: 2.7 x the rate of the fp32 matrix instruction.
// Rows that share a key / value head are packed: row r = g * Lq + i is query i of the g-th head of the group.
#pragma once
#include "common.h"

namespace xattn {

enum { F32 = 0, BF16 = 1, F16 = 2 };

struct Args {
    const void *q, *k, *v, *dout;
    const uint8_t* pad;                                  // [B] rows of Lk bytes, nonzero: not a key
    int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, d_b, d_l, d_h, pad_b;     // strides in elements
    int B, Lq, Lk, H, Hkv, G, D, R;                      // R = G * Lq rows per (batch element, key / value head)
    float scale, c;                                      // c = scale * log2(e)
    int tiles, nsplit, span;                             // row (key) tiles, splits of the other axis, its elements per split
    void* o;                                             // (B, Lq, H, D)
    float* o32;                                          // the same before its rounding, or NULL
    float* lse;                                          // [B Hkv][R] log2 of the row's sum of exponentials; +inf: a row without keys
    float *part, *part2, *part_lse;                      // [nsplit][...] partial results
    float* delta;                                        // [B Hkv][R] <dout, o>
    void *dq, *dk, *dv;
};

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef float fx2 __attribute__((ext_vector_type(2)));
typedef float fx4 __attribute__((ext_vector_type(4)));
typedef unsigned ux4 __attribute__((ext_vector_type(4)));

template <int TY> struct Ty {
    static constexpr int PL = TY == F32 ? 3 : 1;         // planes of an operand
    static constexpr int ES = TY == F32 ? 4 : 2;         // bytes of an element
    static constexpr int EPC = 16 / ES;                  // elements of a 16-byte chunk
    // fp16 keeps 5 exponent bits: probabilities (<= 1) are formed times 2^15, so that one of 2^-29 is still a normal number
    static constexpr float PSHIFT = TY == F16 ? 15.f : 0.f;
};

template <int PL> struct Frag { s16x8 p[PL]; };

template <int TY>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (TY == F16) return __builtin_bit_cast(unsigned, __builtin_convertvector((fx2){a, b}, h16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector((fx2){a, b}, b16x2));
}
template <int TY>
__device__ __forceinline__ fx2 unpack2(unsigned u) {
    if constexpr (TY == F16) return __builtin_convertvector(__builtin_bit_cast(h16x2, u), fx2);
    else return (fx2){__builtin_bit_cast(float, u << 16), __builtin_bit_cast(float, u & 0xffff0000u)};
}
// x = hi + mid + lo, each rounded to nearest bf16.  An infinity stays in the first plane alone.
__device__ __forceinline__ void split2(float a, float b, unsigned& hi, unsigned& mid, unsigned& lo) {
    hi = pack2<BF16>(a, b);
    const fx2 h = unpack2<BF16>(hi);
    const float ra = __builtin_isinf(h.x) ? 0.f : a - h.x, rb = __builtin_isinf(h.y) ? 0.f : b - h.y;
    mid = pack2<BF16>(ra, rb);
    const fx2 m = unpack2<BF16>(mid);
    lo = pack2<BF16>(ra - m.x, rb - m.y);
}
// eight floats -> the planes of a fragment
template <int TY>
__device__ __forceinline__ Frag<Ty<TY>::PL> make_frag(const float* f) {
    Frag<Ty<TY>::PL> r;
    if constexpr (TY == F32) {
        ux4 h, m, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned a, b, c;
            split2(f[2 * i], f[2 * i + 1], a, b, c);
            h[i] = a; m[i] = b; l[i] = c;
        }
        r.p[0] = __builtin_bit_cast(s16x8, h);
        r.p[1] = __builtin_bit_cast(s16x8, m);
        r.p[2] = __builtin_bit_cast(s16x8, l);
    } else {
        ux4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = pack2<TY>(f[2 * i], f[2 * i + 1]);
        r.p[0] = __builtin_bit_cast(s16x8, h);
    }
    return r;
}
template <int TY>
__device__ __forceinline__ f32x16 mma1(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (TY == F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
template <int TY>
__device__ __forceinline__ f32x16 mma(const Frag<Ty<TY>::PL>& a, const Frag<Ty<TY>::PL>& b, f32x16 c) {
    if constexpr (TY == F32) {                           // smallest products first
        c = mma1<TY>(a.p[2], b.p[0], c);
        c = mma1<TY>(a.p[0], b.p[2], c);
        c = mma1<TY>(a.p[1], b.p[1], c);
        c = mma1<TY>(a.p[1], b.p[0], c);
        c = mma1<TY>(a.p[0], b.p[1], c);
        c = mma1<TY>(a.p[0], b.p[0], c);
        return c;
    } else {
        return mma1<TY>(a.p[0], b.p[0], c);
    }
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// the other half's value of the same row (lanes l and l ^ 32 hold the two halves of a score column)
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- LDS tiles: PL planes of ROWS rows of DP + 8 16-bit values.  The 16 bytes behind each row put the rows that one phase of a 128-bit
// read touches on different banks (row stride 4 * odd dwords). -----------------------------------------------------------------------
template <int DP> constexpr int row_len() { return DP + 8; }
template <int TY, int DP, int ROWS> constexpr int tile_len() { return Ty<TY>::PL * ROWS * row_len<DP>(); }   // in 16-bit values

// A operand, rows as they are: lane l holds row row0 + l % 32, columns col0 + 8 (l / 32) + 0..7
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> row_frag(const short* t, int row0, int col0, int lane) {
    Frag<Ty<TY>::PL> f;
    const short* p = t + (row0 + (lane & 31)) * row_len<DP>() + col0 + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) f.p[i] = *reinterpret_cast<const s16x8*>(p + i * ROWS * row_len<DP>());
    return f;
}
// A operand, transposed: lane l holds column col0 + l % 32, contraction slot j = row row0 + 8 (j / 4) + 4 (l / 32) + j % 4
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> col_frag(short* t, int row0, int col0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    Frag<Ty<TY>::PL> f;
    short* p = t + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * row_len<DP>() + col0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) {
        short* pi = p + i * ROWS * row_len<DP>();
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)pi);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(pi + 8 * row_len<DP>()));
        f.p[i] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
}

// ---- staging: ROWS x DP elements through registers, NT threads, 16-byte chunks ---------------------------------------------------------
template <int TY, int DP, int ROWS, int NT> struct Stage {
    static constexpr int CPR = DP / Ty<TY>::EPC;         // chunks of a row
    static constexpr int N = (ROWS * CPR + NT - 1) / NT; // chunks of a thread
    ux4 r[N];
    // row_ptr(row) -> pointer to the row's elements or NULL (zeros instead)
    template <typename F>
    __device__ __forceinline__ void load(int tid, int D, F row_ptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = tid + i * NT, row = id / CPR, col = (id % CPR) * Ty<TY>::EPC;
            ux4 x = {0u, 0u, 0u, 0u};
            if (row < ROWS && col < D) {
                const char* p = row_ptr(row);
                if (p) x = *reinterpret_cast<const ux4*>(p + (size_t)col * Ty<TY>::ES);
            }
            r[i] = x;
        }
    }
    // keep(row): false writes zeros, so that what stands in a padded row (an infinity, a NaN) reaches no product
    template <typename F>
    __device__ __forceinline__ void store(short* t, int tid, F keep) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = tid + i * NT, row = id / CPR, col = (id % CPR) * Ty<TY>::EPC;
            if (ROWS * CPR % NT && row >= ROWS) continue;
            const bool kp = keep(row);
            ux4 x = r[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = kp ? x[j] : 0u;
            short* p = t + row * row_len<DP>() + col;
            if constexpr (TY == F32) {
                unsigned h0, m0, l0, h1, m1, l1;
                const fx4 f = __builtin_bit_cast(fx4, x);
                split2(f.x, f.y, h0, m0, l0);
                split2(f.z, f.w, h1, m1, l1);
                constexpr int PS = ROWS * row_len<DP>();
                *reinterpret_cast<uint2*>(p) = make_uint2(h0, h1);
                *reinterpret_cast<uint2*>(p + PS) = make_uint2(m0, m1);
                *reinterpret_cast<uint2*>(p + 2 * PS) = make_uint2(l0, l1);
            } else {
                *reinterpret_cast<ux4*>(p) = x;
            }
        }
    }
};

// B operand of one row straight from memory: columns 16 s + 8 (l / 32) + 0..7 of every step s; p == NULL or columns behind D: zeros
template <int TY, int DP>
__device__ __forceinline__ void load_row(const void* p, int D, int lane, float (&f)[DP / 16][8]) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int col = 16 * s + 8 * (lane >> 5);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[s][j] = 0.f;
        if (p && col < D) {
            if constexpr (TY == F32) {
                const fx4 a = reinterpret_cast<const fx4*>(p)[col / 4], b = reinterpret_cast<const fx4*>(p)[col / 4 + 1];
#pragma unroll
                for (int j = 0; j < 4; ++j) { f[s][j] = a[j]; f[s][4 + j] = b[j]; }
            } else {
                const ux4 u = reinterpret_cast<const ux4*>(p)[col / 8];
#pragma unroll
                for (int j = 0; j < 4; ++j) { const fx2 w = unpack2<TY>(u[j]); f[s][2 * j] = w.x; f[s][2 * j + 1] = w.y; }
            }
        }
    }
}

// four consecutive elements
template <int TY>
__device__ __forceinline__ void put4(void* p, int64_t e, float a, float b, float c, float d) {
    if constexpr (TY == F32) *reinterpret_cast<fx4*>(reinterpret_cast<float*>(p) + e) = (fx4){a, b, c, d};
    else *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p) + e) = make_uint2(pack2<TY>(a, b), pack2<TY>(c, d));
}

// (batch element, key / value head) bh, packed row r -> element offset of its query in a tensor with the given strides
__device__ __forceinline__ int64_t row_at(const Args& a, int bh, int r, int64_t sb, int64_t sl, int64_t sh) {
    const int b = bh / a.Hkv, kv = bh % a.Hkv, g = r / a.Lq, i = r - g * a.Lq;
    return b * sb + i * sl + (int64_t)(kv * a.G + g) * sh;
}
__device__ __forceinline__ int64_t out_at(const Args& a, int bh, int r) {
    return row_at(a, bh, r, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D);
}

// one behind the last key of [k0, k1) that is not padding (k0: there is none); every thread gets it.  `red`: one int of LDS.
template <int NT>
__device__ __forceinline__ int last_key(const uint8_t* pad, int k0, int k1, int tid, int* red) {
    if (!pad) return k1;
    if (tid == 0) *red = k0;
    __syncthreads();
    int last = k0;
    for (int j = k0 + tid; j < k1; j += NT) last = pad[j] ? last : j + 1;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
    if ((tid & 63) == 0) atomicMax(red, last);
    __syncthreads();
    last = *red;
    __syncthreads();
    return last;
}

// -------------------------------------------------------------------------------------------------------------------------------------
// Forward.  KEYW = false: 4 waves of 32 QS rows each share 64 keys a tile.  KEYW = true, for few rows: one 32-row tile per workgroup,
// each wave takes 32 other keys of the tile and the waves' results are joined at the end.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP, int QS, bool KEYW> struct FwdCfg {
    static constexpr int NW = KEYW && TY == F32 && DP > 64 ? 2 : 4;        // fp32 of 96, 128 columns: the planes of 128 keys do not fit
    static constexpr int NT = 64 * NW;
    static constexpr int ROWS = KEYW ? 32 : 32 * QS * NW;
    static constexpr int BK = KEYW ? 32 * NW : 64;
    static constexpr int KS = KEYW ? 1 : 2;
    static constexpr int TILE = tile_len<TY, DP, BK>();
    static constexpr int RED = KEYW ? NW * DP * 32 * 2 : 0;               // joined results (fp32, in 16-bit units), over the tiles
    static constexpr int LEN = 2 * TILE > RED ? 2 * TILE : RED;
    static constexpr size_t LDS = LEN * 2 + 64 * 4 * NW + 16;
};

template <int TY, int DP, int QS, bool KEYW>
__global__ __launch_bounds__((FwdCfg<TY, DP, QS, KEYW>::NT)) void fwd_kernel(const Args a) {
    using C = FwdCfg<TY, DP, QS, KEYW>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const kt = lds;
    short* const vt = lds + C::TILE;
    float* const stat = reinterpret_cast<float*>(lds + C::LEN);            // [2][NW][32] maxima, sums (KEYW)
    int* const red = reinterpret_cast<int*>(stat + 64 * C::NW);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles; id /= a.tiles;
    const int split = id % a.nsplit, bh = id / a.nsplit;
    const int b = bh / a.Hkv, kv = bh % a.Hkv;
    const char* const kp = (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES;
    const char* const vp = (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES;
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    const int k0 = split * a.span, kend = last_key<C::NT>(pad, k0, min(a.Lk, k0 + a.span), tid, red);

    int row[QS];
    Frag<T::PL> qf[QS][DP / 16];
#pragma unroll
    for (int u = 0; u < QS; ++u) {
        row[u] = tile * C::ROWS + (KEYW ? 0 : 32 * QS * w) + 32 * u + (lane & 31);
        float f[DP / 16][8];
        load_row<TY, DP>(row[u] < a.R ? (const char*)a.q + row_at(a, bh, row[u], a.q_b, a.q_l, a.q_h) * T::ES : nullptr, a.D, lane, f);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) qf[u][s] = make_frag<TY>(f[s]);
    }
    f32x16 o[QS][DP / 32];
    float m[QS], l[QS];
#pragma unroll
    for (int u = 0; u < QS; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.f;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) o[u][t] = zero16();
    }

    Stage<TY, DP, C::BK, C::NT> sk, sv;
    unsigned char pb[(C::BK + 63) / 64];
    const auto fetch = [&](int key) {
        sk.load(tid, a.D, [&](int r) { return key + r < kend ? kp + (int64_t)(key + r) * a.k_l * T::ES : nullptr; });
        sv.load(tid, a.D, [&](int r) { return key + r < kend ? vp + (int64_t)(key + r) * a.v_l * T::ES : nullptr; });
#pragma unroll
        for (int i = 0; i < (C::BK + 63) / 64; ++i) {
            const int j = key + 64 * i + lane;
            pb[i] = j < kend ? (pad ? pad[j] : 0) : 1;
        }
    };
    if (k0 < kend) fetch(k0);
    for (int key = k0; key < kend; key += C::BK) {
        unsigned long long word[(C::BK + 63) / 64];                        // bit j: key j of the tile takes part
#pragma unroll
        for (int i = 0; i < (C::BK + 63) / 64; ++i) word[i] = __builtin_amdgcn_ballot_w64(pb[i] == 0);
        const auto keep = [&](int r) { return (bool)((C::BK > 64 && r >= 64 ? word[(C::BK + 63) / 64 - 1] >> (r - 64) : word[0] >> (r & 63)) & 1ull); };
        __syncthreads();
        sk.store(kt, tid, keep);
        sv.store(vt, tid, keep);
        __syncthreads();
        if (key + C::BK < kend) fetch(key + C::BK);

        const int sub0 = KEYW ? w : 0;                                     // this wave's first group of 32 keys
        f32x16 s[QS][C::KS];
#pragma unroll
        for (int t = 0; t < C::KS; ++t) {
#pragma unroll
            for (int u = 0; u < QS; ++u) s[u][t] = zero16();
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                const Frag<T::PL> kf = row_frag<TY, DP, C::BK>(kt, 32 * (sub0 + t), 16 * d, lane);
#pragma unroll
                for (int u = 0; u < QS; ++u) s[u][t] = mma<TY>(kf, qf[u][d], s[u][t]);
            }
            const unsigned wd = (unsigned)(word[(sub0 + t) >> 1] >> (32 * ((sub0 + t) & 1)));
            if (wd != 0xffffffffu) {
                const unsigned mine = wd >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int u = 0; u < QS; ++u) s[u][t][i] = mine >> (8 * (i >> 2) + (i & 3)) & 1u ? s[u][t][i] : -INFINITY;
            }
        }
        Frag<T::PL> pf[QS][2 * C::KS];
#pragma unroll
        for (int u = 0; u < QS; ++u) {
            float mx = s[u][0][0];
#pragma unroll
            for (int t = 0; t < C::KS; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][t][i]);
            mx = fmaxf(m[u], fmaxf(mx, other_half(mx)));
            if (__builtin_amdgcn_ballot_w64(mx > m[u])) {                  // the running maximum grew somewhere in this wave
                const float f = mx > m[u] ? exp2_f((m[u] - mx) * a.c) : 1.f;
                l[u] *= f;
#pragma unroll
                for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[u][t][i] *= f;
                m[u] = mx;
            }
            const float sh = T::PSHIFT - (m[u] == -INFINITY ? 0.f : m[u] * a.c);
#pragma unroll
            for (int t = 0; t < C::KS; ++t) {
                float p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = exp2_f(fmaf(s[u][t][i], a.c, sh));
                    l[u] += p[i];
                }
                pf[u][2 * t] = make_frag<TY>(p);
                pf[u][2 * t + 1] = make_frag<TY>(p + 8);
            }
        }
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int j = 0; j < 2 * C::KS; ++j) {
                const Frag<T::PL> vf = col_frag<TY, DP, C::BK>(vt, 32 * sub0 + 16 * j, 32 * t, lane);
#pragma unroll
                for (int u = 0; u < QS; ++u) o[u][t] = mma<TY>(vf, pf[u][j], o[u][t]);
            }
    }

    if constexpr (KEYW) {
        // join the waves: row statistics first, then each wave's scaled accumulators through LDS
        float lt = l[0] + other_half(l[0]);
        if (half == 0) {
            stat[w * 32 + lane] = m[0];
            stat[(C::NW + w) * 32 + lane] = lt;
        }
        __syncthreads();                                                    // also: every wave is done with the tiles
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < C::NW; ++i) M = fmaxf(M, stat[i * 32 + (lane & 31)]);
        const float mr = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < C::NW; ++i) {
            const float x = stat[i * 32 + (lane & 31)];
            L += x == -INFINITY ? 0.f : exp2_f((x - mr) * a.c) * stat[(C::NW + i) * 32 + (lane & 31)];
        }
        const float f = m[0] == -INFINITY ? 0.f : exp2_f((m[0] - mr) * a.c);
        const float inv = L == 0.f ? 0.f : f / L;
        float* acc = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[(w * DP + 32 * t + 8 * (i >> 2) + 4 * half + (i & 3)) * 32 + (lane & 31)] = o[0][t][i] * inv;
        __syncthreads();
        if (w == 0 && half == 0 && row[0] < a.R) {
            const float ls = L == 0.f ? -INFINITY : M * a.c + (__builtin_amdgcn_logf(L) - T::PSHIFT);
            if (a.nsplit > 1) a.part_lse[((int64_t)split * a.B * a.Hkv + bh) * a.R + row[0]] = ls;
            else if (a.lse) a.lse[(int64_t)bh * a.R + row[0]] = L == 0.f ? INFINITY : ls;
        }
        const int nq = a.D / 4;
        for (int e = tid; e < 32 * nq; e += C::NT) {
            const int q = e / nq, d = 4 * (e % nq), r = tile * 32 + q;
            if (r >= a.R) continue;
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < C::NW; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] += acc[(i * DP + d + j) * 32 + q];
            if (a.nsplit > 1) {
                put4<F32>(a.part, (((int64_t)split * a.B * a.Hkv + bh) * a.R + r) * a.D + d, x[0], x[1], x[2], x[3]);
            } else {
                const int64_t at = out_at(a, bh, r) + d;
                put4<TY>(a.o, at, x[0], x[1], x[2], x[3]);
                if (a.o32) put4<F32>(a.o32, at, x[0], x[1], x[2], x[3]);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < QS; ++u) {
            const float L = l[u] + other_half(l[u]);
            const float inv = L == 0.f ? 0.f : 1.f / L;
            if (row[u] >= a.R) continue;
            const float ls = L == 0.f ? -INFINITY : m[u] * a.c + (__builtin_amdgcn_logf(L) - T::PSHIFT);
            const int64_t flat = ((int64_t)split * a.B * a.Hkv + bh) * a.R + row[u];
            if (half == 0) {
                if (a.nsplit > 1) a.part_lse[flat] = ls;
                else if (a.lse) a.lse[(int64_t)bh * a.R + row[u]] = L == 0.f ? INFINITY : ls;
            }
            const int64_t at = a.nsplit > 1 ? flat * a.D : out_at(a, bh, row[u]);
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * t + 8 * g;
                    if (d >= a.D) continue;
                    const float x0 = o[u][t][4 * g] * inv, x1 = o[u][t][4 * g + 1] * inv, x2 = o[u][t][4 * g + 2] * inv,
                                x3 = o[u][t][4 * g + 3] * inv;
                    if (a.nsplit > 1) {
                        put4<F32>(a.part, at + d + 4 * half, x0, x1, x2, x3);
                    } else {
                        put4<TY>(a.o, at + d + 4 * half, x0, x1, x2, x3);
                        if (a.o32) put4<F32>(a.o32, at + d + 4 * half, x0, x1, x2, x3);
                    }
                }
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------------------------
// fp16 gradients of scores: p (dp - delta) has the range of dout times v, which 5 exponent bits need not hold.  Each lane keeps a power
// of two for its accumulator column: the largest value seen is brought to 2^10 and the accumulators are rescaled when a later tile
// exceeds 2^14.  It starts at 2^120, so that the first value sets it.  (bf16 and the three-plane form have fp32's exponents: factor 1.)
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int NACC> struct DsScale {
    float f = TY == F16 ? 0x1p120f : 1.f;
    __device__ __forceinline__ void fit(float (&ds)[16], f32x16 (&acc)[NACC]) {
        if constexpr (TY == F16) {
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(ds[i]));
            mx = fmaxf(mx, other_half(mx));
            if (__builtin_amdgcn_ballot_w64(mx * f > 16384.f)) {
                if (mx * f > 16384.f) {
                    const float nf = __builtin_ldexpf(1.f, max(-120, 10 - __builtin_amdgcn_frexp_expf(mx)));
                    const float g = nf / f;                                // both powers of two, nf < f
#pragma unroll
                    for (int t = 0; t < NACC; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[t][i] *= g;
                    f = nf;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] *= f;
        }
    }
};

// -------------------------------------------------------------------------------------------------------------------------------------
// Backward, queries: delta = <dout, o>, dq = scale sum_j p (dp - delta) k.  4 waves of 32 rows, 64 keys a tile: scores and dp
// transposed as in the forward pass (K and V rows are A operands), dq^T accumulates K^T ds^T.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP> struct DqCfg {
    static constexpr int BK = 64, NT = 256, ROWS = 128;
    static constexpr int TILE = tile_len<TY, DP, BK>();
    static constexpr size_t LDS = 2 * TILE * 2 + 16;
};

template <int TY, int DP>
__global__ __launch_bounds__(256) void bwd_dq_kernel(const Args a) {
    using C = DqCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const kt = lds;
    short* const vt = lds + C::TILE;
    int* const red = reinterpret_cast<int*>(lds + 2 * C::TILE);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles; id /= a.tiles;
    const int split = id % a.nsplit, bh = id / a.nsplit;
    const int b = bh / a.Hkv, kv = bh % a.Hkv;
    const char* const kp = (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES;
    const char* const vp = (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES;
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    const int k0 = split * a.span, kend = last_key<C::NT>(pad, k0, min(a.Lk, k0 + a.span), tid, red);

    const int row = tile * C::ROWS + 32 * w + (lane & 31);
    const bool in = row < a.R;
    Frag<T::PL> qf[DP / 16], df[DP / 16];
    float delta = 0.f;
    {
        float f[DP / 16][8];
        load_row<TY, DP>(in ? (const char*)a.q + row_at(a, bh, row, a.q_b, a.q_l, a.q_h) * T::ES : nullptr, a.D, lane, f);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) qf[s] = make_frag<TY>(f[s]);
        float g[DP / 16][8];
        load_row<TY, DP>(in ? (const char*)a.dout + row_at(a, bh, row, a.d_b, a.d_l, a.d_h) * T::ES : nullptr, a.D, lane, f);
        load_row<F32, DP>(in ? a.o32 + out_at(a, bh, row) : nullptr, a.D, lane, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            df[s] = make_frag<TY>(f[s]);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta = fmaf(f[s][j], g[s][j], delta);
        }
        delta += other_half(delta);
    }
    const float ls = (in ? a.lse[(int64_t)bh * a.R + row] : INFINITY) - T::PSHIFT;
    if (split == 0 && half == 0 && in) a.delta[(int64_t)bh * a.R + row] = delta;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();
    DsScale<TY, DP / 32> sc;

    Stage<TY, DP, C::BK, C::NT> sk, sv;
    unsigned char pb;
    const auto fetch = [&](int key) {
        sk.load(tid, a.D, [&](int r) { return key + r < kend ? kp + (int64_t)(key + r) * a.k_l * T::ES : nullptr; });
        sv.load(tid, a.D, [&](int r) { return key + r < kend ? vp + (int64_t)(key + r) * a.v_l * T::ES : nullptr; });
        const int j = key + lane;
        pb = j < kend ? (pad ? pad[j] : 0) : 1;
    };
    if (k0 < kend) fetch(k0);
    for (int key = k0; key < kend; key += C::BK) {
        const unsigned long long word = __builtin_amdgcn_ballot_w64(pb == 0);
        const auto keep = [&](int r) { return (bool)(word >> r & 1ull); };
        __syncthreads();
        sk.store(kt, tid, keep);
        sv.store(vt, tid, keep);
        __syncthreads();
        if (key + C::BK < kend) fetch(key + C::BK);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const unsigned wd = (unsigned)(word >> (32 * t));
            if (wd == 0) continue;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma<TY>(row_frag<TY, DP, C::BK>(kt, 32 * t, 16 * d, lane), qf[d], s);
                dp = mma<TY>(row_frag<TY, DP, C::BK>(vt, 32 * t, 16 * d, lane), df[d], dp);
            }
            float ds[16];
            const unsigned mine = wd >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = exp2_f(fmaf(s[i], a.c, -ls));
                ds[i] = p * (dp[i] - delta);
            }
            if (wd != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = mine >> (8 * (i >> 2) + (i & 3)) & 1u ? ds[i] : 0.f;
            }
            sc.fit(ds, acc);
            const Frag<T::PL> f0 = make_frag<TY>(ds), f1 = make_frag<TY>(ds + 8);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                acc[d] = mma<TY>(col_frag<TY, DP, C::BK>(kt, 32 * t, 32 * d, lane), f0, acc[d]);
                acc[d] = mma<TY>(col_frag<TY, DP, C::BK>(kt, 32 * t + 16, 32 * d, lane), f1, acc[d]);
            }
        }
    }
    if (!in) return;
    const float inv = __builtin_ldexpf(a.scale, -(int)T::PSHIFT) / sc.f;
    const int64_t at = a.nsplit > 1 ? (int64_t)split * a.B * a.Lq * a.H * a.D + out_at(a, bh, row) : out_at(a, bh, row);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * t + 8 * g;
            if (d >= a.D) continue;
            const float x0 = acc[t][4 * g] * inv, x1 = acc[t][4 * g + 1] * inv, x2 = acc[t][4 * g + 2] * inv, x3 = acc[t][4 * g + 3] * inv;
            if (a.nsplit > 1) put4<F32>(a.part, at + d + 4 * half, x0, x1, x2, x3);
            else put4<TY>(a.dq, at + d + 4 * half, x0, x1, x2, x3);
        }
}

// -------------------------------------------------------------------------------------------------------------------------------------
// Backward, keys and values: 4 waves of 32 keys; the packed rows (all heads of the group, all queries) are streamed, 64 a tile.  Here a
// lane owns a KEY: dk^T += Q^T ds, dv^T += dO^T p.  A padded key's column touches no other, so its result is simply written as zeros.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP> struct DkvCfg {
    static constexpr int BR = 64, NT = 256, KEYS = 128;
    static constexpr int TILE = tile_len<TY, DP, BR>();
    static constexpr size_t LDS = 2 * TILE * 2 + 2 * BR * 4 + 16;
};

template <int TY, int DP>
__global__ __launch_bounds__(256) void bwd_dkv_kernel(const Args a) {
    using C = DkvCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const qt = lds;
    short* const dt = lds + C::TILE;
    float* const lsd = reinterpret_cast<float*>(lds + 2 * C::TILE);        // [64] log-sums, [64] deltas of the tile's rows
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tile = id % a.tiles; id /= a.tiles;
    const int split = id % a.nsplit, bh = id / a.nsplit;
    const int b = bh / a.Hkv, kv = bh % a.Hkv;
    const int key = tile * C::KEYS + 32 * w + (lane & 31);
    const bool in = key < a.Lk, live = in && !(a.pad && a.pad[b * a.pad_b + key]);
    const bool work = __builtin_amdgcn_ballot_w64(live) != 0;             // of this wave
    const int r0 = split * a.span, rend = __syncthreads_or(work) ? min(a.R, r0 + a.span) : r0;

    Frag<T::PL> kf[DP / 16], vf[DP / 16];
    {
        float f[DP / 16][8];
        load_row<TY, DP>(live ? (const char*)a.k + (b * a.k_b + key * a.k_l + kv * a.k_h) * T::ES : nullptr, a.D, lane, f);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) kf[s] = make_frag<TY>(f[s]);
        load_row<TY, DP>(live ? (const char*)a.v + (b * a.v_b + key * a.v_l + kv * a.v_h) * T::ES : nullptr, a.D, lane, f);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) vf[s] = make_frag<TY>(f[s]);
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dk[t] = dv[t] = zero16();
    DsScale<TY, DP / 32> sc;

    Stage<TY, DP, C::BR, C::NT> sq, sd;
    float st = 0.f;
    const char* const qb = (const char*)a.q + (b * a.q_b + (int64_t)kv * a.G * a.q_h) * T::ES;
    const char* const db = (const char*)a.dout + (b * a.d_b + (int64_t)kv * a.G * a.d_h) * T::ES;
    const auto fetch = [&](int r) {
        const int g0 = r / a.Lq, i0 = r - g0 * a.Lq;                       // uniform
        const auto at = [&](int x, const char* base, int64_t sl, int64_t sh) -> const char* {
            if (r + x >= rend) return nullptr;
            int g = g0, i = i0 + x;
            if (i >= a.Lq) { g += i / a.Lq; i %= a.Lq; }
            return base + (i * sl + g * sh) * T::ES;
        };
        sq.load(tid, a.D, [&](int x) { return at(x, qb, a.q_l, a.q_h); });
        sd.load(tid, a.D, [&](int x) { return at(x, db, a.d_l, a.d_h); });
        const int x = r + (tid & 63);
        if (tid < 64) st = x < rend ? a.lse[(int64_t)bh * a.R + x] - T::PSHIFT : INFINITY;
        else if (tid < 128) st = x < rend ? a.delta[(int64_t)bh * a.R + x] : 0.f;
    };
    if (r0 < rend) fetch(r0);
    for (int r = r0; r < rend; r += C::BR) {
        __syncthreads();
        sq.store(qt, tid, [](int) { return true; });
        sd.store(dt, tid, [](int) { return true; });
        if (tid < 128) lsd[tid] = st;
        __syncthreads();
        if (r + C::BR < rend) fetch(r + C::BR);
        if (!work) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (r + 32 * t >= rend) continue;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma<TY>(row_frag<TY, DP, C::BR>(qt, 32 * t, 16 * d, lane), kf[d], s);
                dp = mma<TY>(row_frag<TY, DP, C::BR>(dt, 32 * t, 16 * d, lane), vf[d], dp);
            }
            float p[16], ds[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const fx4 ls = *reinterpret_cast<const fx4*>(lsd + 32 * t + 8 * g + 4 * half);
                const fx4 de = *reinterpret_cast<const fx4*>(lsd + 64 + 32 * t + 8 * g + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[4 * g + i] = exp2_f(fmaf(s[4 * g + i], a.c, -ls[i]));
                    ds[4 * g + i] = p[4 * g + i] * (dp[4 * g + i] - de[i]);
                }
            }
            sc.fit(ds, dk);
            const Frag<T::PL> p0 = make_frag<TY>(p), p1 = make_frag<TY>(p + 8), d0 = make_frag<TY>(ds), d1 = make_frag<TY>(ds + 8);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                dv[d] = mma<TY>(col_frag<TY, DP, C::BR>(dt, 32 * t, 32 * d, lane), p0, dv[d]);
                dk[d] = mma<TY>(col_frag<TY, DP, C::BR>(qt, 32 * t, 32 * d, lane), d0, dk[d]);
                dv[d] = mma<TY>(col_frag<TY, DP, C::BR>(dt, 32 * t + 16, 32 * d, lane), p1, dv[d]);
                dk[d] = mma<TY>(col_frag<TY, DP, C::BR>(qt, 32 * t + 16, 32 * d, lane), d1, dk[d]);
            }
        }
    }
    if (!in) return;
    const float ik = live ? __builtin_ldexpf(a.scale, -(int)T::PSHIFT) / sc.f : 0.f, iv = __builtin_ldexpf(1.f, -(int)T::PSHIFT);
    const int64_t at = (((int64_t)(a.nsplit > 1 ? split : 0) * a.B + b) * a.Lk + key) * a.Hkv * a.D + (int64_t)kv * a.D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * t + 8 * g;
            if (d >= a.D) continue;
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = live ? dk[t][4 * g + i] * ik : 0.f;                 // a select: a padded key's column may hold NaN
                y[i] = live ? dv[t][4 * g + i] * iv : 0.f;
            }
            if (a.nsplit > 1) {
                put4<F32>(a.part, at + d + 4 * half, x[0], x[1], x[2], x[3]);
                put4<F32>(a.part2, at + d + 4 * half, y[0], y[1], y[2], y[3]);
            } else {
                put4<TY>(a.dk, at + d + 4 * half, x[0], x[1], x[2], x[3]);
                put4<TY>(a.dv, at + d + 4 * half, y[0], y[1], y[2], y[3]);
            }
        }
}

// ---- joining splits -------------------------------------------------------------------------------------------------------------------
// forward: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max); a thread owns four columns of a row
template <int TY>
__global__ __launch_bounds__(256) void join_fwd_kernel(const Args a) {
    const int nq = a.D / 4;
    const int64_t rows = (int64_t)a.B * a.Hkv * a.R, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * nq) return;
    const int64_t fr = e / nq;
    const int d = 4 * (int)(e % nq);
    float M = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, a.part_lse[s * rows + fr]);
    const float mr = M == -INFINITY ? 0.f : M;
    float W = 0.f;
    fx4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
        const float wgt = exp2_f(a.part_lse[s * rows + fr] - mr);
        const fx4 y = *reinterpret_cast<const fx4*>(a.part + (s * rows + fr) * a.D + d);
        W += wgt;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(wgt, y[j], x[j]);
    }
    const float inv = W == 0.f ? 0.f : 1.f / W;
    const int bh = (int)(fr / a.R), r = (int)(fr % a.R);
    const int64_t at = out_at(a, bh, r) + d;
    put4<TY>(a.o, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (a.o32) put4<F32>(a.o32, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (d == 0 && a.lse) a.lse[fr] = W == 0.f ? INFINITY : M + __builtin_amdgcn_logf(W);
}
// backward: out[i] = sum_s part[s][i], s ascending; n a multiple of 4
template <int TY>
__global__ __launch_bounds__(256) void join_sum_kernel(const float* part, void* out, int64_t n, int nsplit) {
    const int64_t e = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (e >= n) return;
    fx4 x = *reinterpret_cast<const fx4*>(part + e);
    for (int s = 1; s < nsplit; ++s) {
        const fx4 y = *reinterpret_cast<const fx4*>(part + s * n + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += y[j];
    }
    put4<TY>(out, e, x[0], x[1], x[2], x[3]);
}

// ---- launches of one element type (defined in that type's unit) -------------------------------------------------------------------------
template <int TY> int launch_fwd(const Args& a, int keyw, int qs, hipStream_t s);
template <int TY> int launch_join_fwd(const Args& a, hipStream_t s);
template <int TY> int launch_bwd_dq(const Args& a, hipStream_t s);
template <int TY> int launch_bwd_dkv(const Args& a, hipStream_t s);
template <int TY> int launch_join_sum(const float* part, void* out, int64_t n, int nsplit, hipStream_t s);

}  // namespace xattn
