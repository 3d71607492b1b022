// Cross attention: queries of one sequence against keys / values of another one, softmax(scale q k^T) v per head, with a key padding
// mask, shared key / value heads and the backward pass.  Included by one unit per element type (xattn_f32 / _bf16 / _f16.hip) and by the
// host side (xattn.hip).
//
// One pass over the keys with a running maximum and sum (no score matrix in memory).  Every product is a 32x32x16 16-bit MFMA:
//   * the streamed operand (K, V forward and dQ; Q, dO for dK / dV) is staged row-major in LDS; as an MFMA A operand its rows are read
//     with ds_read_b128, transposed with ds_read_b64_tr_b16 (4 rows x 16 columns per 16 lanes), both without bank conflicts (swizzle());
//   * the stationary operand sits in registers as B operand, so that a score tile comes out TRANSPOSED: lane l owns query (or key)
//     l % 32 and holds 16 scores of it.  Row statistics are per-lane scalars (one lane exchange per tile), and the tile's registers are,
//     packed, the B operand of the next product: contraction slot (l / 32, j) of step s is row 16 s + 8 (j / 4) + 4 (l / 32) + j % 4 of
//     the tile, and the transposed LDS read delivers the same order.  Probabilities never pass through LDS.
//   * fp32 elements are split into three bf16 planes (24 significand bits, fp32's exponent range) and multiplied with six products, the
//     dropped ones are below 2^-24 of the operands' product: 2.7 x the rate of the fp32 matrix instruction.
//   * 16-bit elements: probabilities, and score gradients backward, are rounded to the element type for the second product: one MFMA
//     instead of the two that a second plane would take, for half a step of the type per probability (results are then off by about 1.4
//     times what the rounding of the result alone costs).  The forward forms of up to 64 rows are bound by the keys' bytes and have the time
//     for that second plane, so a row among few is rounded once only.  Sums, maxima, log-sums and accumulators are fp32.
// Rows that share a key / value head are packed: row r = g * Lq + i is query i of the g-th head of the group.
// Times at the kernels below are the kernel's alone, between the slowest and the fastest card measured; rates count 4, 6 and 8 D
// operations a score for the forward pass, dq, and dk and dv.
#pragma once
#include <type_traits>

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
    // Forward, the running maximum follows only when a row's scores exceed it by 2^LAZY: p <= 2^LAZY, few rescalings.
    // fp16 keeps 5 exponent bits.  Backward, probabilities (<= 1) are formed times 2^15, so that one of 2^-29 is still a normal number;
    // forward they are formed times 2^13, so that one of 2^-27 of the row's largest is, and below that each is off by up to 2^-38 of the
    // largest.  (2^8 and 2^7 left 2^-21, and a row whose largest probability meets a value near 0 lost up to four bits of its result.)
    static constexpr float PSHIFT = TY == F16 ? 15.f : 0.f;
    static constexpr float LAZY = TY == F16 ? 2.f : 8.f;
    static constexpr float FSHIFT = TY == F16 ? 15.f - LAZY : 0.f;
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
// x = hi + mid + lo, each rounded to nearest bf16; values beyond bf16's largest have that one as hi, and the planes still add up to them.
// An infinity stands in the last plane alone: mma() multiplies that plane by the other operand's first one only, which has its value's sign
// and is 0 where the value is, so the product is the infinity (or the NaN) of the definition.  In the first plane it would also meet the
// other's lower planes, whose signs say nothing.  PLAIN: values that are neither (probabilities; tiles that were looked through).
constexpr float MOST = 0x1.fep127f;
template <bool PLAIN = false>
__device__ __forceinline__ void split2(float a, float b, unsigned& hi, unsigned& mid, unsigned& lo) {
    const bool ia = !PLAIN && __builtin_isinf(a), ib = !PLAIN && __builtin_isinf(b);
    hi = PLAIN ? pack2<BF16>(a, b)
              : pack2<BF16>(__builtin_amdgcn_fmed3f(ia ? 0.f : a, -MOST, MOST), __builtin_amdgcn_fmed3f(ib ? 0.f : b, -MOST, MOST));
    const fx2 h = unpack2<BF16>(hi);
    const float ra = ia ? 0.f : a - h.x, rb = ib ? 0.f : b - h.y;          // a NaN gets here, whatever the median made of it
    mid = pack2<BF16>(ra, rb);
    const fx2 m = unpack2<BF16>(mid);
    lo = pack2<BF16>(ia ? a : ra - m.x, ib ? b : rb - m.y);
}
// eight floats -> the planes of a fragment
template <int TY, bool PLAIN = false>
__device__ __forceinline__ Frag<Ty<TY>::PL> make_frag(const float* f) {
    Frag<Ty<TY>::PL> r;
    if constexpr (TY == F32) {
        ux4 h, m, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned a, b, c;
            split2<PLAIN>(f[2 * i], f[2 * i + 1], a, b, c);
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

// a value that is the same for all lanes, in a scalar register: quotients are computed by the vector unit, and a buffer descriptor that
// depends on one would be looped over
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// 0, which the compiler does not know: a second pass whose bounds contain it shares no addresses with the first, and its registers hold none
// for it (fwd_token_kernel and its join, fp16, 4 x 8 heads of 4 rows x 30011 keys x 128 columns: 94.5 -> 92.5 us)
__device__ __forceinline__ int hidden_zero() {
    int z = 0;
    asm volatile("" : "+s"(z));
    return z;
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

// ---- LDS tiles: PL planes of ROWS rows of DP 16-bit values, the 16-byte chunks of a row permuted --------------------------------------
// LDS has 64 banks of 4 bytes; a row covers DP / 2 of them.  A 128-bit read serves the same chunk of 16 rows at once (lanes {0-3, 12-15,
// 20-27}, {4-11, 16-19, 28-31} and these + 32), a transposing 64-bit read four chunks of 4 rows (lanes 0-31, 32-63).  Chunk c of row r is
// stored at c ^ swizzle(r), which spreads both over all banks for every DP (rows padded by 16 bytes instead: 2 to 4 lanes a bank on the
// transposed reads).  swizzle(r + 16) == swizzle(r), so a lane's addresses differ by constants between groups of 16 rows.
template <int DP> __device__ __forceinline__ int swizzle(int r) {
    if constexpr (DP == 64) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
    else if constexpr (DP == 128) return (r & 3) << 2 | ((r >> 2) & 3);
    else return (r >> 2) & 3;                            // 32, 96: row starts already differ by quarters of the banks
}
template <int TY, int DP, int ROWS> constexpr int tile_len() { return Ty<TY>::PL * ROWS * DP; }      // in 16-bit values

// A operand, rows as they are: lane l holds row row0 + l % 32, columns col0 + 8 (l / 32) + 0..7
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> row_frag(const short* t, int row0, int col0, int lane) {
    Frag<Ty<TY>::PL> f;
    const int r = lane & 31;
    const short* p = t + r * DP + 8 * ((col0 / 8 + (lane >> 5)) ^ swizzle<DP>(r)) + row0 * DP;
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) f.p[i] = *reinterpret_cast<const s16x8*>(p + i * ROWS * DP);
    return f;
}
// A operand, transposed: lane l holds column col0 + l % 32, contraction slot j = row row0 + 8 (j / 4) + 4 (l / 32) + j % 4
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> col_frag(short* t, int row0, int col0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    Frag<Ty<TY>::PL> f;
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), c = col0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    short* p = t + r * DP + 8 * (c ^ swizzle<DP>(r)) + 4 * (lane & 1) + row0 * DP;
    short* q = t + (r + 8) * DP + 8 * (c ^ swizzle<DP>(r + 8)) + 4 * (lane & 1) + row0 * DP;
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) {
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + i * ROWS * DP));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(q + i * ROWS * DP));
        f.p[i] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
}

// ---- staging: ROWS x DP elements through registers, NT threads, 16-byte chunks ---------------------------------------------------------
// Rows `stride` bytes apart from a wave-uniform base; a lane's offsets are 32 bits (the entry point refuses strides of 2^24 bytes and
// more), rows behind the end and columns behind D read zeros by the buffer's bound.
template <int TY, int DP, int ROWS, int NT> struct Stage {
    static constexpr int CPR = DP / Ty<TY>::EPC;         // chunks of a row
    static constexpr int N = (ROWS * CPR + NT - 1) / NT; // chunks of a thread
    static constexpr bool PART = ROWS * CPR % NT != 0;   // the last one not of every thread
    ux4 r[N];
    __device__ __forceinline__ static int row_of(int tid, int i) { return (tid + i * NT) / CPR; }
    __device__ __forceinline__ static int col_of(int tid, int i) { return (tid + i * NT) % CPR * Ty<TY>::EPC; }
    // rows [0, rows) of the tile exist; rows >= 1.  Chunk i of a thread lies i STEP rows behind its first one: the base moves, its offset stays
    __device__ __forceinline__ void load(int tid, int D, const char* base, int64_t stride, int rows) {
        if constexpr (NT % CPR == 0) {
            constexpr int STEP = NT / CPR;
            // (no branch: one would turn the stride, and with it the descriptors, into lane values)
            const unsigned off = ((unsigned)row_of(tid, 0) * (unsigned)stride + col_of(tid, 0) * Ty<TY>::ES) | (col_of(tid, 0) >= D ? FAVAE_OOB : 0u);
            const int bytes = min(rows, ROWS) * (int)stride, step = STEP * (int)stride;    // under 2^31: at most 128 rows of 2^24 - 16
#pragma unroll
            for (int i = 0; i < N; ++i)
                r[i] = __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(base + i * step, (unsigned)max(bytes - i * step, 0)), off, 0, 0);
        } else {
            const auto rs = make_rsrc(base, (unsigned)min(rows, ROWS) * (unsigned)stride);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const unsigned off = (unsigned)row_of(tid, i) * (unsigned)stride + col_of(tid, i) * Ty<TY>::ES;
                r[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, off | (col_of(tid, i) >= D || (PART && row_of(tid, i) >= ROWS) ? FAVAE_OOB : 0u), 0, 0);
            }
        }
    }
    // any rows: row_ptr(row) -> pointer to the row's elements or NULL (zeros instead)
    template <typename F>
    __device__ __forceinline__ void gather(int tid, int D, F row_ptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            ux4 x = {0u, 0u, 0u, 0u};
            if (col_of(tid, i) < D && (!PART || row_of(tid, i) < ROWS)) {
                const char* p = row_ptr(row_of(tid, i));
                if (p) x = *reinterpret_cast<const ux4*>(p + col_of(tid, i) * Ty<TY>::ES);
            }
            r[i] = x;
        }
    }
    // keep(row): false writes zeros, so that what stands in a padded row (an infinity, a NaN) reaches no product
    template <typename F>
    __device__ __forceinline__ void blank(int tid, F keep) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int row = row_of(tid, i);
            asm volatile("" : "+v"(row));                                  // computed here, where it is seldom needed: no registers in the loop
            const bool kp = (PART && row >= ROWS) || keep(row);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[i][j] = kp ? r[i][j] : 0u;
        }
    }
    // some value of this thread's is finite and of 2^120 or more (fp32, bf16)
    __device__ __forceinline__ bool huge() const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned u = r[i][j];
                any = any || (u & 0x7fffffffu) - 0x7b800000u < 0x04000000u;
                if constexpr (TY == BF16) any = any || (u << 16 & 0x7fffffffu) - 0x7b800000u < 0x04000000u;
            }
        return any;
    }
    __device__ __forceinline__ void store(short* t, int tid) const {
        if constexpr (TY == F32) {                                         // one comparison for all of a wave's values, three instructions less for each
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const fx4 f = __builtin_bit_cast(fx4, r[i]);
                most = fmaxf(fmaxf(fmaxf(most, fabsf(f.x)), fmaxf(fabsf(f.y), fabsf(f.z))), fabsf(f.w));
            }
            if (__builtin_amdgcn_ballot_w64(most > MOST)) put<false>(t, tid);
            else put<true>(t, tid);
        } else {
            put<true>(t, tid);
        }
    }
    template <bool PLAIN>
    __device__ __forceinline__ void put(short* t, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row_of(tid, i), col = col_of(tid, i);
            if (PART && row >= ROWS) continue;
            // chunks a multiple of 16 rows apart: one address and constants
            const int row0 = NT % (16 * CPR) == 0 ? row_of(tid, 0) : row, col0 = NT % (16 * CPR) == 0 ? col_of(tid, 0) : col;
            short* p = t + row0 * DP + 8 * ((col0 / 8) ^ swizzle<DP>(row0)) + (col0 & 7) + (NT % (16 * CPR) == 0 ? i * (NT / CPR) * DP : 0);
            if constexpr (TY == F32) {
                unsigned h0, m0, l0, h1, m1, l1;
                const fx4 f = __builtin_bit_cast(fx4, r[i]);
                split2<PLAIN>(f.x, f.y, h0, m0, l0);
                split2<PLAIN>(f.z, f.w, h1, m1, l1);
                constexpr int PS = ROWS * DP;
                *reinterpret_cast<uint2*>(p) = make_uint2(h0, h1);
                *reinterpret_cast<uint2*>(p + PS) = make_uint2(m0, m1);
                *reinterpret_cast<uint2*>(p + 2 * PS) = make_uint2(l0, l1);
            } else {
                *reinterpret_cast<ux4*>(p) = r[i];
            }
        }
    }
};

// B operand of one row straight from memory: columns 16 s + 8 (l / 32) + 0..7 of every step s; p == NULL or columns behind D: zeros
template <int DP>
__device__ __forceinline__ void load_floats(const float* p, int D, int lane, float (&f)[DP / 16][8]) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int col = 16 * s + 8 * (lane >> 5);
        fx4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (p && col < D) {
            a = reinterpret_cast<const fx4*>(p)[col / 4];
            b = reinterpret_cast<const fx4*>(p)[col / 4 + 1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[s][j] = a[j]; f[s][4 + j] = b[j]; }
    }
}
template <int TY, int DP>
__device__ __forceinline__ void load_row(const void* p, int D, int lane, Frag<Ty<TY>::PL> (&r)[DP / 16]) {
    if constexpr (TY == F32) {
        float f[DP / 16][8];
        load_floats<DP>((const float*)p, D, lane, f);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) r[s] = make_frag<TY>(f[s]);
    } else {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int col = 16 * s + 8 * (lane >> 5);
            r[s].p[0] = (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
            if (p && col < D) r[s].p[0] = reinterpret_cast<const s16x8*>(p)[col / 8];
        }
    }
}
// element j of a fragment as a float (the three planes add up to it exactly)
template <int TY> __device__ __forceinline__ float frag_at(const Frag<Ty<TY>::PL>& f, int j) {
    float x = 0.f;
#pragma unroll
    for (int i = Ty<TY>::PL - 1; i >= 0; --i) {
        const short e = f.p[i][j];
        x += unpack2<TY>((unsigned)(unsigned short)e).x;
    }
    return x;
}

// what eight floats lose in the 16-bit fragment made of them, as a fragment
template <int TY> __device__ __forceinline__ Frag<Ty<TY>::PL> rest_frag(const float* x, const Frag<Ty<TY>::PL>& f) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = x[j] - frag_at<TY>(f, j);
    return make_frag<TY>(r);
}

// a 16-bit fragment with zeros for infinities and NaN: the values that the second plane of the probabilities meets.  That plane is 0 or has
// any sign, where the first one alone gives an infinite value's product.  (All exponent bits plus one step carry into the sign bit.)
template <int TY, bool CARE> __device__ __forceinline__ Frag<Ty<TY>::PL> finite_frag(const Frag<Ty<TY>::PL>& f) {
    if constexpr (!CARE) return f;
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    constexpr unsigned EXP = TY == F16 ? 0x7c007c00u : 0x7f807f80u, ONE = TY == F16 ? 0x04000400u : 0x00800080u;
    ux4 u = __builtin_bit_cast(ux4, f.p[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] &= ~__builtin_bit_cast(unsigned, __builtin_bit_cast(s16x2, (u[i] & EXP) + ONE) >> 15);
    Frag<Ty<TY>::PL> r;
    r.p[0] = __builtin_bit_cast(s16x8, u);
    return r;
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
// A wave's 32 packed rows from the wave-uniform r0 on: where they are of one head, which the longer axis makes the rule, row r0 + x lies
// x strides behind the first (the division that finds the head is then made once for all 32, by scalars).
struct Rows {
    int r0;
    int64_t first;                                       // element of row r0, or -1: several heads (or rows behind the last)
    __device__ __forceinline__ Rows(const Args& a, int bh, int r, int64_t sb, int64_t sl, int64_t sh) {
        r0 = __builtin_amdgcn_readfirstlane(r);
        const int g = uniform(r0 / a.Lq), i = r0 - g * a.Lq;
        first = r0 + 32 <= a.R && i + 32 <= a.Lq ? bh / a.Hkv * sb + i * sl + (int64_t)(bh % a.Hkv * a.G + g) * sh : -1;
    }
    __device__ __forceinline__ bool has(const Args& a, int x) const { return first >= 0 || r0 + x < a.R; }
    // has(x)
    __device__ __forceinline__ int64_t at(const Args& a, int bh, int x, int64_t sb, int64_t sl, int64_t sh) const {
        return first >= 0 ? first + (unsigned)x * (unsigned)sl : row_at(a, bh, r0 + x, sb, sl, sh);
    }
};
// a lane's row, r0 + lane % 32, of a tensor of TY; NULL behind the last one
template <int TY>
__device__ __forceinline__ const char* lane_row(const Args& a, const void* p, int bh, int r0, int lane, int64_t sb, int64_t sl, int64_t sh) {
    const Rows rows(a, bh, r0, sb, sl, sh);
    return rows.has(a, lane & 31) ? (const char*)p + rows.at(a, bh, lane & 31, sb, sl, sh) * Ty<TY>::ES : nullptr;
}
struct OutRows : Rows {
    __device__ __forceinline__ OutRows(const Args& a, int bh, int r) : Rows(a, bh, r, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D) {}
    __device__ __forceinline__ int64_t at(const Args& a, int bh, int x) const {
        return Rows::at(a, bh, x, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D);
    }
};

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
    last = __builtin_amdgcn_readfirstlane(*red);
    __syncthreads();
    return last;
}

// two LDS buffers (one barrier a tile) where as many workgroups still fit a CU as its registers allow
constexpr int bufs_of(int tile, int waves, bool pre) { return pre && 4 * tile * 2 <= (waves == 1 ? 150000 : 77000) ? 2 : 1; }
// keys of a tile that take part: bit j of word i is key 64 i + j.  The mask's bytes come a tile ahead, a byte a lane.
template <int BK> struct KeyBits {
    static constexpr int N = (BK + 63) / 64;
    static constexpr unsigned long long ALL = BK >= 64 ? ~0ull : (1ull << (BK & 63)) - 1;
    unsigned b[N];
    __device__ __forceinline__ void load(const uint8_t* pad, int key, int kend, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            b[i] = 0;
            if (pad) b[i] = __builtin_amdgcn_raw_buffer_load_b8(make_rsrc(pad + key + 64 * i, (unsigned)uniform(max(0, min(64, kend - key - 64 * i)))), lane, 0, 0);
        }
    }
    __device__ __forceinline__ bool words(int left, unsigned long long (&word)[N]) const {      // left: keys from the tile's first on
        bool all = true;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = min(left - 64 * i, min(64, BK - 64 * i));
            word[i] = n <= 0 ? 0ull : __builtin_amdgcn_ballot_w64(b[i] == 0) & (~0ull >> (64 - n));
            all = all && word[i] == ALL;
        }
        return all;
    }
};

// A pass over the keys that ends with a sum which is no finite number is made once more, with care:
//   * the sums of probabilities times values are divided at the end, so they leave 32 bits where values times the number of keys (times
//     2^LAZY) exceed 3.4e38, although the result does not: probabilities are formed times SMALL (fp16 values are below 2^16 and need none);
//   * where 16-bit probabilities have a second plane (few rows), it meets zeros for infinities (finite_frag);
//   * c s - c m is one multiply-add with a rounded c m, half a step of which is a factor of 2^8 for c m = 2^33 (and of fp16's range for 2^26):
//     rows of such maxima take c (s - m) (Ref).  Then the sum of a row's probabilities may be 0, too, although it has keys.
// All leave the bits of everything that was a number.
template <int TY> constexpr float SMALL = TY == F16 ? 1.f : 0x1p-40f;
template <int TY, bool CARE> __device__ __forceinline__ float prob(float x) { return CARE ? exp2_f(x) * SMALL<TY> : exp2_f(x); }
// A row whose probabilities sum to 0 has no keys, and gives zeros, or keys whose scores are all -infinity, and gives the NaN of the formula
// (an infinite query makes one of every score that is not).  A split writes zeros for both, and NO_SCORE as the second one's log-sum.
constexpr float NO_SCORE = -3.402823466e38f;
__device__ __forceinline__ float no_sum(bool keys) { return keys ? __builtin_nanf("") : 0.f; }
__device__ __forceinline__ float no_lse(bool keys) { return keys ? __builtin_nanf("") : INFINITY; }
// whether any of the first NW waves says so, to all threads; `flags`: NW ints of LDS.  One barrier: every wave is done with the tiles, too.
template <int NW> __device__ __forceinline__ bool some_wave(bool mine, int w, int lane, int* flags) {
    const bool any = __builtin_amdgcn_ballot_w64(mine) != 0;
    if (w < NW && lane == 0) flags[w] = any;
    __syncthreads();
    int r = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) r |= flags[i];
    return uniform(r) != 0;
}
// the exponent of a row's probabilities is c (s - r) + sh
struct Ref {
    float r, sh;
    __device__ __forceinline__ Ref(float m, float c, float shift, bool care) {
        r = care && fabsf(m * c) > 0x1p20f && fabsf(m) < INFINITY ? m : 0.f;
        sh = shift - (m == -INFINITY || r != 0.f ? 0.f : m * c);
    }
};
template <int N, typename V> __device__ __forceinline__ bool not_finite(const V (&o)[N]) {
    float z = 0.f;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / 4); ++i) z = fmaf(o[t][i], 0.f, z);
    return !(z == 0.f);
}

// key masks: a tile's scores start at 0 for a key and at -infinity for padding, as the accumulator of their first product
__device__ __forceinline__ f32x16 start16(const float* bias, int half) {
    f32x16 s;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const fx4 x = *reinterpret_cast<const fx4*>(bias + 8 * g + 4 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g + i] = x[i];
    }
    return s;
}
template <int TY, int DP, int ROWS, bool ALL>
__device__ __forceinline__ f32x16 scores(const short* t, int row0, const Frag<Ty<TY>::PL> (&b)[DP / 16], const float* bias, int lane) {
    f32x16 s;
    if constexpr (ALL) s = zero16();
    else s = start16(bias, lane >> 5);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) s = mma<TY>(row_frag<TY, DP, ROWS>(t, row0, 16 * d, lane), b[d], s);
    return s;
}

// -------------------------------------------------------------------------------------------------------------------------------------
// Forward: m = running maximum of s = q k^T, l = sum 2^(c s - c m), o = sum 2^(c s - c m) v / l.
// KEYW = false: 4 waves of 32 rows each share 64 keys a tile (fp32: 32, its planes are three times as large).  KEYW = true, for 17 to 64
// rows: one 32-row tile per workgroup, each wave takes 32 other keys of the tile and the waves' results are joined at the end.
// Bound by issue: a 32 x 32 tile of 64 columns is 8 MFMAs and per lane 16 exponentials, multiply-adds, maxima / 2 and sums and 8 packings;
// beside them addresses, waits and what a wave does once cost as much again, so every instruction counts (descriptors in scalars instead
// of lane values: 118 -> 107 us).  bf16, 64 heads x 4096 rows x 1024 keys x 64 columns: 95-118 us, 580-720 TFLOP/s.  fp32 is bound by its
// six products: 16 heads x 2048 x 2048 x 128 in two spans 181-196 us, 175-190 TFLOP/s, six times that on the matrix pipe; 10 us to join.
// One 32-row group a wave, 3 waves a SIMD with 16-bit elements of up to 64 columns (V's first half is read ahead of the exponentials: 3 %).
// 64 rows a wave took the same time, two groups with interleaved exponentials 10 % more, four waves (32 keys at a time) 6 %, the next
// tile's stores between the products 15 %, sums by products with ones 4 %.  fp32 of 128 columns spills 24 registers (72 bytes of scratch a
// lane; six loads of it a tile of 96 MFMAs); the other forms spill none.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP, bool KEYW> struct FwdCfg {
    static constexpr int NT = 256;
    static constexpr int NW = KEYW && TY == F32 && DP > 64 ? 2 : 4;        // waves that compute: the planes of 128 keys of 96, 128 fp32 columns
    static constexpr int ROWS = KEYW ? 32 : 32 * NW;                       // do not fit LDS, there two waves only load
    static constexpr bool PRE = !(TY == F32 && DP > 64 && !KEYW);         // the next tile is loaded under this one's products (registers allowing)
    static constexpr int WAVES = KEYW && (TY == F32 ? DP > 64 : DP == 128) ? 1 : !KEYW && TY != F32 && DP <= 64 ? 3 : 2;       // a SIMD; also keeps accumulators out of the second register file
    static constexpr int BK = KEYW ? 32 * NW : TY == F32 ? 32 : 64;
    static constexpr int KS = KEYW ? 1 : BK / 32;
    static constexpr int TILE = tile_len<TY, DP, BK>();
    static constexpr int BUFS = bufs_of(TILE, WAVES, PRE);
    static constexpr int RED = KEYW ? NW * DP * 32 * 2 : 0;               // joined results (fp32, in 16-bit units), over the tiles
    static constexpr int LEN = 2 * TILE * BUFS > RED ? 2 * TILE * BUFS : RED;
    static constexpr size_t LDS = LEN * 2 + BUFS * BK * 4 + 64 * 4 * NW + 4 * 4;
};

template <int TY, int DP, bool KEYW>
__global__ __launch_bounds__((FwdCfg<TY, DP, KEYW>::NT), (FwdCfg<TY, DP, KEYW>::WAVES)) void fwd_kernel(const Args a) {
    using C = FwdCfg<TY, DP, KEYW>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    float* const bias = reinterpret_cast<float*>(lds + C::LEN);           // [BUFS][BK]
    float* const stat = bias + C::BUFS * C::BK;                           // [2][NW][32] maxima, sums (KEYW)
    int* const red = reinterpret_cast<int*>(stat + 64 * C::NW);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    // workgroups of one head follow one another on an XCD: its keys stay in that L2.  Few rows share nothing (each split reads its own
    // keys), there the heads of a ragged batch alternate instead.
    int id = KEYW ? blockIdx.x : xcd_remap(blockIdx.x, gridDim.x);
    const int heads = a.B * a.Hkv;
    const int bh = uniform(KEYW ? id % heads : id / (a.tiles * a.nsplit));
    id = KEYW ? id / heads : id % (a.tiles * a.nsplit);
    const int split = uniform(id / a.tiles), tile = uniform(id % a.tiles);
    const int b = uniform(bh / a.Hkv), kv = bh - b * a.Hkv;
    const char* const kp = (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES;
    const char* const vp = (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES;
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    const int k0 = split * a.span;
    int kend = min(a.Lk, k0 + a.span);

    Stage<TY, DP, C::BK, C::NT> sk, sv;
    KeyBits<C::BK> pb;
    const auto fetch = [&](int key) {
        sk.load(tid, a.D, kp + key * a.k_l * T::ES, a.k_l * T::ES, kend - key);
        sv.load(tid, a.D, vp + key * a.v_l * T::ES, a.v_l * T::ES, kend - key);
        pb.load(pad, key, kend, lane);
    };
    if (C::PRE) fetch(k0);                                                 // k0 < Lk; on its way while the mask is looked through
    const int row0 = tile * C::ROWS + (KEYW ? 0 : 32 * w), row = row0 + (lane & 31);
    Frag<T::PL> qf[DP / 16];
    load_row<TY, DP>(lane_row<TY>(a, a.q, bh, row0, lane, a.q_b, a.q_l, a.q_h), a.D, lane, qf);
    kend = last_key<C::NT>(pad, k0, kend, tid, red);
    f32x16 o[DP / 32];
    float m, l, up = 1.f;                                                  // up: what brings l back to its size
    int buf = 0;
    const auto pass = [&](auto care) {
        constexpr bool CARE = decltype(care)::value;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) o[t] = zero16();
        for (int key = k0; key < kend; key += C::BK) {
            if (!C::PRE) fetch(key);
            unsigned long long word[KeyBits<C::BK>::N];
            const bool all = pb.words(kend - key, word);
            short* const kt = lds + buf * 2 * C::TILE;
            short* const vt = kt + C::TILE;
            float* const bi = bias + buf * C::BK;
            if (C::BUFS == 1) __syncthreads();
            if (!all) {
                const auto keep = [&](int r) { return (bool)((C::BK > 64 && r >= 64 ? word[KeyBits<C::BK>::N - 1] >> (r & 63) : word[0] >> (r & 63)) & 1ull); };
                sk.blank(tid, keep);
                sv.blank(tid, keep);
                if (tid < C::BK) bi[tid] = keep(tid) ? 0.f : -INFINITY;
            }
            sk.store(kt, tid);
            sv.store(vt, tid);
            __syncthreads();
            if (C::PRE && key + C::BK < kend) fetch(key + C::BK);
            if (C::BUFS == 2) buf ^= 1;

            const int sub0 = KEYW ? w : 0;                                     // this wave's first group of 32 keys
            if (KEYW && w >= C::NW) continue;
            f32x16 s[C::KS];
            if (all) {
#pragma unroll
                for (int t = 0; t < C::KS; ++t) s[t] = scores<TY, DP, C::BK, true>(kt, 32 * (sub0 + t), qf, bi, lane);
            } else {
#pragma unroll
                for (int t = 0; t < C::KS; ++t) s[t] = scores<TY, DP, C::BK, false>(kt, 32 * (sub0 + t), qf, bi + 32 * (sub0 + t), lane);
            }
            constexpr bool AHEAD = !KEYW && TY != F32 && DP <= 64;
            Frag<T::PL> vf[2 * C::KS];
            if constexpr (AHEAD) {
#pragma unroll
                for (int j = 0; j < 2 * C::KS; ++j) vf[j] = col_frag<TY, DP, C::BK>(vt, 16 * j, 0, lane);
                __builtin_amdgcn_sched_barrier(0);
            }
            float mx = s[0][0];
#pragma unroll
            for (int t = 0; t < C::KS; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
            mx = fmaxf(mx, other_half(mx));
            if (__builtin_amdgcn_ballot_w64((mx - m) * a.c > T::LAZY)) {       // some row of this wave outgrew its maximum
                const float to = fmaxf(m, mx), f = to > m ? exp2_f((m - to) * a.c) : 1.f;
                l *= f;
#pragma unroll
                for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][i] *= f;
                m = to;
            }
            const Ref ref(m, a.c, T::FSHIFT, CARE);
            Frag<T::PL> pf[2 * C::KS];
#pragma unroll
            for (int t = 0; t < C::KS; ++t) {
                float p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = prob<TY, CARE>(fmaf(CARE ? s[t][i] - ref.r : s[t][i], a.c, ref.sh));
                    l += p[i];
                }
                pf[2 * t] = make_frag<TY, true>(p);
                pf[2 * t + 1] = make_frag<TY, true>(p + 8);
                if constexpr (KEYW && TY != F32) {                             // few rows: the matrix pipe has time for what p loses in 16 bits
                    const Frag<T::PL> r0 = rest_frag<TY>(p, pf[0]), r1 = rest_frag<TY>(p + 8, pf[1]);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) {
                        o[d] = mma<TY>(finite_frag<TY, CARE>(col_frag<TY, DP, C::BK>(vt, 32 * sub0, 32 * d, lane)), r0, o[d]);
                        o[d] = mma<TY>(finite_frag<TY, CARE>(col_frag<TY, DP, C::BK>(vt, 32 * sub0 + 16, 32 * d, lane)), r1, o[d]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int j = 0; j < 2 * C::KS; ++j) {
                    if constexpr (AHEAD) {
                        o[t] = mma<TY>(vf[j], pf[j], o[t]);
                        if (t + 1 < DP / 32) {
                            vf[j] = col_frag<TY, DP, C::BK>(vt, 16 * j, 32 * (t + 1), lane);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    } else {
                        o[t] = mma<TY>(col_frag<TY, DP, C::BK>(vt, 32 * sub0 + 16 * j, 32 * t, lane), pf[j], o[t]);
                    }
                }
        }
    };
    pass(std::false_type{});
    float lt;
    const auto odd = [&] {                                                  // KEYW: the waves are joined, row statistics first
        lt = l + other_half(l);
        if (KEYW && half == 0 && w < C::NW) {
            stat[w * 32 + lane] = m;
            stat[(C::NW + w) * 32 + lane] = lt;
        }
        return some_wave<C::NW>(not_finite(o) || (lt == 0.f && m > -INFINITY), w, lane, red);
    };
    if (__builtin_expect(odd(), 0)) {
        const int z = hidden_zero();
        kend += z;
        if (C::PRE) fetch(k0 + z);
        pass(std::true_type{});
        up = 1.f / SMALL<TY>;
        odd();
    }
    if constexpr (KEYW) {
        // each wave's scaled accumulators through LDS
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < C::NW; ++i) M = fmaxf(M, stat[i * 32 + (lane & 31)]);
        const float mr = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < C::NW; ++i) {
            const float x = stat[i * 32 + (lane & 31)];
            L += x == -INFINITY ? 0.f : exp2_f((x - mr) * a.c) * stat[(C::NW + i) * 32 + (lane & 31)];
        }
        const float f = m == -INFINITY ? 0.f : exp2_f((m - mr) * a.c);
        const float inv = L == 0.f ? no_sum(kend > k0 && a.nsplit == 1) : f / L;
        float* acc = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (w < C::NW) acc[(w * DP + 32 * t + 8 * (i >> 2) + 4 * half + (i & 3)) * 32 + (lane & 31)] = o[t][i] * inv;
        __syncthreads();
        if (w == 0 && half == 0 && row < a.R) {
            const float ls = L == 0.f ? (kend > k0 ? NO_SCORE : -INFINITY) : M * a.c + (__builtin_amdgcn_logf(L * up) - T::FSHIFT);
            if (a.nsplit > 1) a.part_lse[((int64_t)split * a.B * a.Hkv + bh) * a.R + row] = ls;
            else if (a.lse) a.lse[(int64_t)bh * a.R + row] = L == 0.f ? no_lse(kend > k0) : ls;
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
        const float inv = lt == 0.f ? no_sum(kend > k0 && a.nsplit == 1) : 1.f / lt;
        const float ls = lt == 0.f ? (kend > k0 ? NO_SCORE : -INFINITY) : m * a.c + (__builtin_amdgcn_logf(lt * up) - T::FSHIFT);
        const int64_t flat = ((int64_t)split * a.B * a.Hkv + bh) * a.R + row;
        const bool in = row < a.R;
        const OutRows to_row(a, bh, row0);
        if (half == 0 && in) {
            if (a.nsplit > 1) a.part_lse[flat] = ls;
            else if (a.lse) a.lse[(int64_t)bh * a.R + row] = lt == 0.f ? no_lse(kend > k0) : ls;
        }
        // 32-bit results: a lane's four consecutive columns are one 16-byte store
        if (TY == F32 || a.nsplit > 1 || a.o32) {
            float* const to = a.nsplit > 1 ? a.part : TY == F32 ? (float*)a.o : a.o32;
            const int64_t at = a.nsplit > 1 ? flat * a.D : in ? to_row.at(a, bh, lane & 31) : 0;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * t + 8 * g;
                    if (d < a.D && in) put4<F32>(to, at + d + 4 * half, o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv);
                }
        }
        // 16-bit results: transposed through LDS (a wave's own 32 rows), so that eight lanes or more write a row's consecutive 16 bytes
        if constexpr (TY != F32) {
            if (a.nsplit > 1) return;
            __syncthreads();                                                // every wave is done with the tiles
            static_assert(4 * 32 * DP <= C::LEN, "the waves' rows fit");
            short* const mine = lds + w * 32 * DP;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int r = lane & 31, c = 4 * t + g;
                    *reinterpret_cast<uint2*>(mine + r * DP + 8 * (c ^ swizzle<DP>(r)) + 4 * half) =
                        make_uint2(pack2<TY>(o[t][4 * g] * inv, o[t][4 * g + 1] * inv), pack2<TY>(o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv));
                }
            __syncthreads();
            constexpr int CPR = DP / 8;
#pragma unroll
            for (int i = 0; i < 32 * CPR / 64; ++i) {
                const int e = lane + 64 * i, r = e / CPR, c = e % CPR;
                if (to_row.has(a, r) && 8 * c < a.D)
                    *reinterpret_cast<ux4*>((short*)a.o + to_row.at(a, bh, r) + 8 * c) = *reinterpret_cast<const ux4*>(mine + r * DP + 8 * (c ^ swizzle<DP>(r)));
            }
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------------------------
// Forward over few keys (a prompt): all of them stay in LDS and a workgroup goes through many row tiles, each wave by itself without a
// barrier, the next tile's queries on their way.  One maximum per row, nothing is rescaled.  What is left is reading q and writing o.
// bf16 and fp16, 128 heads x 4096 rows x 77 keys x 64 columns: 33 us, 4.1 TB/s of q and o (fwd_kernel: 46); fp32, 256 heads x 256 x 77 x 64:
// 22 us, there each wave has one row tile and waits for the keys' planes.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP> struct ShortCfg {
    static constexpr int NT = 256, KEYS = TY == F32 ? 96 : 128, KT = KEYS / 32;
    static constexpr bool OK = TY != F32 || DP <= 64;                      // two workgroups a CU
    static constexpr int TILE = tile_len<TY, DP, KEYS>();
    static constexpr int OUT = TY == F32 || DP == 128 ? 0 : 4 * 32 * DP;   // 16-bit results on their way out, a wave's own 32 rows (128: no room)
    static constexpr size_t LDS = (2 * TILE + OUT) * 2 + KEYS * 4 + 16;
};

template <int TY, int DP>
__global__ __launch_bounds__(256, 2) void fwd_short_kernel(const Args a) {
    using C = ShortCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const kt = lds;
    short* const vt = lds + C::TILE;
    short* const out = lds + 2 * C::TILE;
    float* const bias = reinterpret_cast<float*>(out + C::OUT);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int id = xcd_remap(blockIdx.x, gridDim.x), bh = uniform(id / a.tiles), b = uniform(bh / a.Hkv), kv = bh - b * a.Hkv;
    const int r0 = (id - bh * a.tiles) * a.span, rend = min(a.R, r0 + a.span);  // this workgroup's rows; span is a multiple of 128
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    bool huge = false, keys;                                               // keys: there is one that is not padding
    {
        Stage<TY, DP, C::KEYS, C::NT> sk, sv;
        sk.load(tid, a.D, (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES, a.k_l * T::ES, a.Lk);
        sv.load(tid, a.D, (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES, a.v_l * T::ES, a.Lk);
        const bool k0 = lane < a.Lk && !(pad && pad[lane]), k1 = 64 + lane < a.Lk && !(pad && pad[64 + lane]);
        const unsigned long long w0 = __builtin_amdgcn_ballot_w64(k0), w1 = __builtin_amdgcn_ballot_w64(k1);
        keys = (w0 | w1) != 0;
        const auto keep = [&](int r) { return (bool)((r >= 64 ? w1 >> (r & 63) : w0 >> r) & 1ull); };
        sk.blank(tid, keep);
        sv.blank(tid, keep);
        sk.store(kt, tid);
        sv.store(vt, tid);
        if (tid < C::KEYS) bias[tid] = keep(tid) ? 0.f : -INFINITY;
        if constexpr (TY != F16) huge = sv.huge();
    }
    // Probabilities are at most 1: fp16 takes them times 2^15.  Their sums with values of 2^120 and more could leave 32 bits before they are
    // divided: there they are formed times 2^-16 (and their exponents' argument is rounded at 2^-20, which is why not everywhere).
    float shift = T::PSHIFT;
    if constexpr (TY == F16) __syncthreads();
    else if (uniform(__syncthreads_or(huge))) shift = -16.f;
    // groups of 32 keys; behind the last key: bias -infinity.  Without keys there is no group: a query of NaN makes NaN scores of padding, too
    const int nk = keys ? (a.Lk + 31) / 32 : 0;

    const auto row_ptr = [&](int rt) { return rt < rend ? lane_row<TY>(a, a.q, bh, rt, lane, a.q_b, a.q_l, a.q_h) : nullptr; };
    Frag<T::PL> qf[DP / 16];
    load_row<TY, DP>(row_ptr(r0 + 32 * w), a.D, lane, qf);
    for (int rt = r0 + 32 * w; rt < rend; rt += 128) {
        const int row = rt + (lane & 31);
        const bool in = row < rend;
        f32x16 s[C::KT];
#pragma unroll
        for (int t = 0; t < C::KT; ++t)
            if (t < nk) s[t] = scores<TY, DP, C::KEYS, false>(kt, 32 * t, qf, bias + 32 * t, lane);
        load_row<TY, DP>(row_ptr(rt + 128), a.D, lane, qf);               // the next tile's, under what follows
        float m = -INFINITY;
#pragma unroll
        for (int t = 0; t < C::KT; ++t)
            if (t < nk) {
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, s[t][i]);
            }
        m = fmaxf(m, other_half(m));
        const Ref ref(m, a.c, shift, true);
        if (__builtin_amdgcn_ballot_w64(ref.r != 0.f)) {
#pragma unroll
            for (int t = 0; t < C::KT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] -= ref.r;
        }
        float l = 0.f;
        f32x16 o[DP / 32];
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) o[t] = zero16();
#pragma unroll
        for (int t = 0; t < C::KT; ++t)
            if (t < nk) {
                float p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = exp2_f(fmaf(s[t][i], a.c, ref.sh));
                    l += p[i];
                }
                const Frag<T::PL> p0 = make_frag<TY, true>(p), p1 = make_frag<TY, true>(p + 8);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    o[d] = mma<TY>(col_frag<TY, DP, C::KEYS>(vt, 32 * t, 32 * d, lane), p0, o[d]);
                    o[d] = mma<TY>(col_frag<TY, DP, C::KEYS>(vt, 32 * t + 16, 32 * d, lane), p1, o[d]);
                }
            }
        l += other_half(l);
        const float inv = l == 0.f ? no_sum(keys) : 1.f / l;
        const OutRows to_row(a, bh, rt);
        if (half == 0 && in && a.lse) a.lse[(int64_t)bh * a.R + row] = l == 0.f ? no_lse(keys) : m * a.c + (__builtin_amdgcn_logf(l) - shift);
        if (TY == F32 || a.o32) {
            float* const to = TY == F32 ? (float*)a.o : a.o32;
            const int64_t at = in ? to_row.at(a, bh, lane & 31) : 0;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * t + 8 * g;
                    if (d < a.D && in) put4<F32>(to, at + d + 4 * half, o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv);
                }
        }
        if constexpr (TY != F32 && C::OUT == 0) {
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * t + 8 * g;
                    if (d < a.D && in)
                        put4<TY>(a.o, to_row.at(a, bh, lane & 31) + d + 4 * half, o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv);
                }
        } else if constexpr (TY != F32) {
            short* const mine = out + w * 32 * DP;
            __builtin_amdgcn_wave_barrier();                               // a wave's LDS accesses are served in order
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int r = lane & 31, c = 4 * t + g;
                    *reinterpret_cast<uint2*>(mine + r * DP + 8 * (c ^ swizzle<DP>(r)) + 4 * half) =
                        make_uint2(pack2<TY>(o[t][4 * g] * inv, o[t][4 * g + 1] * inv), pack2<TY>(o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv));
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            constexpr int CPR = DP / 8;
#pragma unroll
            for (int i = 0; i < 32 * CPR / 64; ++i) {
                const int e = lane + 64 * i, r = e / CPR, c = e % CPR;
                if (to_row.has(a, r) && 8 * c < a.D)
                    *reinterpret_cast<ux4*>((short*)a.o + to_row.at(a, bh, r) + 8 * c) = *reinterpret_cast<const ux4*>(mine + r * DP + 8 * (c ^ swizzle<DP>(r)));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------------------------
// Forward of up to 16 rows a head group (a decoding step): bound by the bytes of K and V.  16x16x32 MFMAs hold the 16 rows in half the
// registers of the 32-row form, so that two workgroups of 128 keys a tile share a CU and one's loads run under the other's arithmetic.
// Each wave takes 32 keys of the tile: lane l holds row l % 16 and keys 4 (l / 16) + i and 16 + 4 (l / 16) + i, which are also the
// contraction slots of the second product.  fp16, 4 x 8 heads of 4 rows x 30011 keys x 128 columns of ragged sequences (400 MB) in 16 spans:
// 88 us, 4.6 TB/s (32-row form: 125), and 5 us for the join; fp32 242 us for 800 MB, 3.3 TB/s, where two of the four waves only load; bf16,
// 256 heads of one row x 77 keys: 6 us, of which a launch and two memory latencies are 4.
// The matrix pipe has time here: probabilities are rounded to two planes, products of both are summed.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY> __device__ __forceinline__ fx4 mma16_1(s16x8 a, s16x8 b, fx4 c) {
    if constexpr (TY == F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
template <int TY>
__device__ __forceinline__ fx4 mma16(const Frag<Ty<TY>::PL>& a, const Frag<Ty<TY>::PL>& b, fx4 c) {
    if constexpr (TY == F32) {
        c = mma16_1<TY>(a.p[2], b.p[0], c);
        c = mma16_1<TY>(a.p[0], b.p[2], c);
        c = mma16_1<TY>(a.p[1], b.p[1], c);
        c = mma16_1<TY>(a.p[1], b.p[0], c);
        c = mma16_1<TY>(a.p[0], b.p[1], c);
        c = mma16_1<TY>(a.p[0], b.p[0], c);
        return c;
    } else {
        return mma16_1<TY>(a.p[0], b.p[0], c);
    }
}
// rows row0 + l % 16, columns 32 s + 8 (l / 16) + 0..7
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> row_frag16(const short* t, int row0, int s, int lane) {
    Frag<Ty<TY>::PL> f;
    const int r = lane & 15;
    const short* p = t + r * DP + 8 * ((4 * s + (lane >> 4)) ^ swizzle<DP>(r)) + row0 * DP;
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) f.p[i] = *reinterpret_cast<const s16x8*>(p + i * ROWS * DP);
    return f;
}
// column col0 + l % 16, slots j = rows row0 + 16 (j / 4) + 4 (l / 16) + j % 4
template <int TY, int DP, int ROWS>
__device__ __forceinline__ Frag<Ty<TY>::PL> col_frag16(short* t, int row0, int col0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    Frag<Ty<TY>::PL> f;
    const int r = 4 * (lane >> 4) + ((lane & 15) >> 2), c = col0 / 8 + ((lane & 3) >> 1);
    short* p = t + r * DP + 8 * (c ^ swizzle<DP>(r)) + 4 * (lane & 1) + row0 * DP;
#pragma unroll
    for (int i = 0; i < Ty<TY>::PL; ++i) {
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + i * ROWS * DP));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + i * ROWS * DP + 16 * DP));
        f.p[i] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
}

template <int TY, int DP> struct TokCfg {
    static constexpr int NT = 256;
    static constexpr int NW = TY == F32 && DP > 64 ? 2 : 4;                // as in FwdCfg
    static constexpr int BK = 32 * NW;
    static constexpr int TILE = tile_len<TY, DP, BK>();
    static constexpr int RED = NW * DP * 16 * 2;
    static constexpr int LEN = 2 * TILE > RED ? 2 * TILE : RED;
    static constexpr size_t LDS = LEN * 2 + BK * 4 + 32 * 4 * NW + 16;
};

template <int TY, int DP>
__global__ __launch_bounds__(256, 2) void fwd_token_kernel(const Args a) {
    using C = TokCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const kt = lds;
    short* const vt = lds + C::TILE;
    float* const bias = reinterpret_cast<float*>(lds + C::LEN);           // [BK]
    float* const stat = bias + C::BK;                                     // [2][NW][16] maxima, sums
    int* const red = reinterpret_cast<int*>(stat + 32 * C::NW);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    const int heads = a.B * a.Hkv, split = uniform(blockIdx.x / heads), bh = blockIdx.x - split * heads;   // heads alternate: a ragged batch is spread evenly
    const int b = uniform(bh / a.Hkv), kv = bh - b * a.Hkv;
    const char* const kp = (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES;
    const char* const vp = (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES;
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    const int k0 = split * a.span;
    int kend = min(a.Lk, k0 + a.span);

    Stage<TY, DP, C::BK, C::NT> sk, sv;
    KeyBits<C::BK> pb;
    const auto fetch = [&](int key) {
        sk.load(tid, a.D, kp + key * a.k_l * T::ES, a.k_l * T::ES, kend - key);
        sv.load(tid, a.D, vp + key * a.v_l * T::ES, a.v_l * T::ES, kend - key);
        pb.load(pad, key, kend, lane);
    };
    fetch(k0);                                                             // k0 < Lk
    const int row = lane & 15;
    Frag<T::PL> qf[DP / 32];
    {
        const char* const q = row < a.R ? (const char*)a.q + row_at(a, bh, row, a.q_b, a.q_l, a.q_h) * T::ES : nullptr;
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) {
            const int col = 32 * s + 8 * quad;
            ux4 x[T::ES / 2] = {};
            if (q && col < a.D) {
#pragma unroll
                for (int i = 0; i < T::ES / 2; ++i) x[i] = reinterpret_cast<const ux4*>(q + col * T::ES)[i];
            }
            if constexpr (TY == F32) {
                float f[8];
                const fx4 lo = __builtin_bit_cast(fx4, x[0]), hi = __builtin_bit_cast(fx4, x[1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) { f[j] = lo[j]; f[4 + j] = hi[j]; }
                qf[s] = make_frag<TY>(f);
            } else {
                qf[s].p[0] = __builtin_bit_cast(s16x8, x[0]);
            }
        }
    }
    kend = last_key<C::NT>(pad, k0, kend, tid, red);
    fx4 o[DP / 16];
    float m, l, up = 1.f;                                                  // up: what brings l back to its size
    const auto pass = [&](auto care) {
        constexpr bool CARE = decltype(care)::value;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] = (fx4){0.f, 0.f, 0.f, 0.f};
        for (int key = k0; key < kend; key += C::BK) {
            unsigned long long word[KeyBits<C::BK>::N];
            const bool all = pb.words(kend - key, word);
            __syncthreads();
            if (!all) {
                const auto keep = [&](int r) { return (bool)((r >= 64 ? word[KeyBits<C::BK>::N - 1] >> (r & 63) : word[0] >> (r & 63)) & 1ull); };
                sk.blank(tid, keep);
                sv.blank(tid, keep);
                if (tid < C::BK) bias[tid] = keep(tid) ? 0.f : -INFINITY;
            }
            sk.store(kt, tid);
            sv.store(vt, tid);
            __syncthreads();
            if (key + C::BK < kend) fetch(key + C::BK);
            if (w >= C::NW) continue;

            fx4 s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[t] = (fx4){0.f, 0.f, 0.f, 0.f};
                if (!all) s[t] = *reinterpret_cast<const fx4*>(bias + 32 * w + 16 * t + 4 * quad);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) s[t] = mma16<TY>(row_frag16<TY, DP, C::BK>(kt, 32 * w + 16 * t, d, lane), qf[d], s[t]);
            }
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(s[0][i], s[1][i]));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__builtin_amdgcn_ballot_w64((mx - m) * a.c > T::LAZY)) {
                const float to = fmaxf(m, mx), f = to > m ? exp2_f((m - to) * a.c) : 1.f;
                l *= f;
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) o[t] *= f;
                m = to;
            }
            const Ref ref(m, a.c, T::FSHIFT, CARE);
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = prob<TY, CARE>(fmaf(CARE ? s[i >> 2][i & 3] - ref.r : s[i >> 2][i & 3], a.c, ref.sh));
                l += p[i];
            }
            const Frag<T::PL> pf = make_frag<TY, true>(p);
            Frag<T::PL> rest;
            if constexpr (TY != F32) rest = rest_frag<TY>(p, pf);              // the matrix pipe has time for what p loses in 16 bits
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                const Frag<T::PL> vf = col_frag16<TY, DP, C::BK>(vt, 32 * w, 16 * t, lane);
                if constexpr (TY != F32) o[t] = mma16<TY>(finite_frag<TY, CARE>(vf), rest, o[t]);
                o[t] = mma16<TY>(vf, pf, o[t]);
            }
        }
    };
    pass(std::false_type{});
    const auto total = [](float x) {
        x += __shfl_xor(x, 16, 64);
        return x + __shfl_xor(x, 32, 64);
    };
    const auto odd = [&] {
        const float lt = total(l);
        if (quad == 0 && w < C::NW) {
            stat[w * 16 + row] = m;
            stat[(C::NW + w) * 16 + row] = lt;
        }
        return some_wave<C::NW>(not_finite(o) || (lt == 0.f && m > -INFINITY), w, lane, red);
    };
    if (__builtin_expect(odd(), 0)) {
        const int z = hidden_zero();
        kend += z;
        fetch(k0 + z);
        pass(std::true_type{});
        up = 1.f / SMALL<TY>;
        odd();
    }
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < C::NW; ++i) M = fmaxf(M, stat[i * 16 + row]);
    const float mr = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < C::NW; ++i) {
        const float x = stat[i * 16 + row];
        L += x == -INFINITY ? 0.f : exp2_f((x - mr) * a.c) * stat[(C::NW + i) * 16 + row];
    }
    const float f = m == -INFINITY ? 0.f : exp2_f((m - mr) * a.c);
    const float inv = L == 0.f ? no_sum(kend > k0 && a.nsplit == 1) : f / L;
    float* acc = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (w < C::NW) acc[(w * DP + 16 * t + 4 * quad + i) * 16 + row] = o[t][i] * inv;
    __syncthreads();
    if (w == 0 && quad == 0 && row < a.R) {
        const float ls = L == 0.f ? (kend > k0 ? NO_SCORE : -INFINITY) : M * a.c + (__builtin_amdgcn_logf(L * up) - T::FSHIFT);
        if (a.nsplit > 1) a.part_lse[((int64_t)split * heads + bh) * a.R + row] = ls;
        else if (a.lse) a.lse[(int64_t)bh * a.R + row] = L == 0.f ? no_lse(kend > k0) : ls;
    }
    const int nq = a.D / 4;
    for (int e = tid; e < a.R * nq; e += C::NT) {
        const int r = e / nq, d = 4 * (e % nq);
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < C::NW; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] += acc[(i * DP + d + j) * 16 + r];
        if (a.nsplit > 1) {
            put4<F32>(a.part, (((int64_t)split * heads + bh) * a.R + r) * a.D + d, x[0], x[1], x[2], x[3]);
        } else {
            const int64_t at = out_at(a, bh, r) + d;
            put4<TY>(a.o, at, x[0], x[1], x[2], x[3]);
            if (a.o32) put4<F32>(a.o32, at, x[0], x[1], x[2], x[3]);
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
// Bound by both pipes: 12 MFMAs beside 16 exponentials, 32 multiply-adds and 8 packings per lane and tile of 64 columns.  bf16, 64 heads x
// 4096 x 1024 x 64: 122-147 us, 700-850 TFLOP/s (both groups of 32 keys in one stretch of code, or dp started at -delta: 8-14 % more, their
// registers cost a wave a SIMD); fp16, 12 key heads x 3063 rows x 515 x 80: 37 us, 288 workgroups on 256 CUs, 80 columns computed as 96;
// fp32, 256 x 256 x 77 x 64: 26 us.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP> struct DqCfg {
    static constexpr int BK = TY == F32 || DP == 128 ? 32 : 64, NT = 256, ROWS = 128;
    static constexpr int WAVES = TY == F32 && DP > 64 ? 1 : 2;
    static constexpr int TILE = tile_len<TY, DP, BK>();
    static constexpr int BUFS = bufs_of(TILE, WAVES, true);
    static constexpr size_t LDS = 2 * TILE * BUFS * 2 + BUFS * BK * 4 + 16;
};

template <int TY, int DP>
__global__ __launch_bounds__(256, (DqCfg<TY, DP>::WAVES)) void bwd_dq_kernel(const Args a) {
    using C = DqCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    float* const bias = reinterpret_cast<float*>(lds + 2 * C::TILE * C::BUFS);
    int* const red = reinterpret_cast<int*>(bias + C::BUFS * C::BK);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int rest = uniform(id / a.tiles), tile = id - rest * a.tiles, bh = uniform(rest / a.nsplit), split = rest - bh * a.nsplit;
    const int b = uniform(bh / a.Hkv), kv = bh - b * a.Hkv;
    const char* const kp = (const char*)a.k + (b * a.k_b + kv * a.k_h) * T::ES;
    const char* const vp = (const char*)a.v + (b * a.v_b + kv * a.v_h) * T::ES;
    const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b : nullptr;
    const int k0 = split * a.span;
    int kend = min(a.Lk, k0 + a.span);

    Stage<TY, DP, C::BK, C::NT> sk, sv;
    KeyBits<C::BK> pb;
    const auto fetch = [&](int key) {
        sk.load(tid, a.D, kp + key * a.k_l * T::ES, a.k_l * T::ES, kend - key);
        sv.load(tid, a.D, vp + key * a.v_l * T::ES, a.v_l * T::ES, kend - key);
        pb.load(pad, key, kend, lane);
    };
    fetch(k0);                                                             // k0 < Lk; on its way while the mask is looked through
    kend = last_key<C::NT>(pad, k0, kend, tid, red);

    const int row0 = tile * C::ROWS + 32 * w, row = row0 + (lane & 31);
    const bool in = row < a.R;
    const OutRows to_row(a, bh, row0);
    Frag<T::PL> qf[DP / 16], df[DP / 16];
    load_row<TY, DP>(lane_row<TY>(a, a.q, bh, row0, lane, a.q_b, a.q_l, a.q_h), a.D, lane, qf);
    load_row<TY, DP>(lane_row<TY>(a, a.dout, bh, row0, lane, a.d_b, a.d_l, a.d_h), a.D, lane, df);
    float delta = 0.f;
    {
        float g[DP / 16][8];
        load_floats<DP>(in ? a.o32 + to_row.at(a, bh, lane & 31) : nullptr, a.D, lane, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) delta = fmaf(frag_at<TY>(df[s], j), g[s][j], delta);
        delta += other_half(delta);
    }
    const float ls = (in ? a.lse[(int64_t)bh * a.R + row] : INFINITY) - T::PSHIFT;
    if (split == 0 && half == 0 && in) a.delta[(int64_t)bh * a.R + row] = delta;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();
    DsScale<TY, DP / 32> sc;

    int buf = 0;
    for (int key = k0; key < kend; key += C::BK) {
        unsigned long long words[1];
        const bool all = pb.words(kend - key, words);
        const unsigned long long word = words[0];
        short* const kt = lds + buf * 2 * C::TILE;
        short* const vt = kt + C::TILE;
        float* const bi = bias + buf * C::BK;
        if (C::BUFS == 1) __syncthreads();
        if (!all) {
            const auto keep = [&](int r) { return (bool)(word >> r & 1ull); };
            sk.blank(tid, keep);
            sv.blank(tid, keep);
            if (tid < C::BK) bi[tid] = keep(tid) ? 0.f : -INFINITY;
        }
        sk.store(kt, tid);
        sv.store(vt, tid);
        __syncthreads();
        if (key + C::BK < kend) fetch(key + C::BK);
        if (C::BUFS == 2) buf ^= 1;
#pragma unroll
        for (int t = 0; t < C::BK / 32; ++t) {
            if ((unsigned)(word >> (32 * t)) == 0) continue;
            f32x16 s, dp;
            const auto both = [&](auto every) {
                s = scores<TY, DP, C::BK, decltype(every)::value>(kt, 32 * t, qf, bi + 32 * t, lane);
                dp = zero16();
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) dp = mma<TY>(row_frag<TY, DP, C::BK>(vt, 32 * t, 16 * d, lane), df[d], dp);
            };
            if (all) both(std::true_type{});
            else both(std::false_type{});
            float ds[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] = exp2_f(fmaf(s[i], a.c, -ls)) * (dp[i] - delta);
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
    const int64_t at = (a.nsplit > 1 ? (int64_t)split * a.B * a.Lq * a.H * a.D : 0) + to_row.at(a, bh, lane & 31);
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
// Bound by the matrix pipe and LDS: 16 MFMAs and 16 KB of LDS reads a wave and tile of 64 columns.  bf16, 64 heads x 4096 x 1024 x 64:
// 144-176 us, 780-950 TFLOP/s (dp started at 0: 10 % more; stores of the next tile between the products: 8 %); fp16, 12 key heads x
// 3063 rows x 515 x 80 in 8 spans: 38 us and 5 for each join; fp32, 256 x 256 x 77 x 64: 37 us.
// -------------------------------------------------------------------------------------------------------------------------------------
template <int TY, int DP> struct DkvCfg {
    static constexpr int BR = TY == F32 || DP > 64 ? 32 : 64, NT = 256, KEYS = 128;
    static constexpr bool TIGHT = DP > 64 || (TY == F32 && DP > 32);
    static constexpr int WAVES = TY == F32 && DP > 64 ? 1 : 2;
    // more than 64 columns (fp32: 32): the values' rows stay in LDS, their operands are read again for every tile, and dp is formed after
    // the probabilities are used; a wave's registers hold no more beside both accumulators.  bf16, 64 heads x 1024 x 1024: 128 columns
    // 148 -> 87 us (790 TFLOP/s, two waves a SIMD instead of one), 96 columns 87 -> 76 us; fp32 the same time within 2 %.  At 128 columns
    // 16-bit elements still spill 8 (bf16) and 12 (fp16) registers, 36 and 52 bytes of scratch that the row loop reads again, and fp32 9
    // into the accumulation registers.
    static constexpr int VALS = TIGHT ? tile_len<TY, DP, KEYS>() : 0;
    static constexpr int TILE = tile_len<TY, DP, BR>();
    static constexpr int BUFS = TIGHT ? 1 : bufs_of(TILE, WAVES, true);
    static constexpr size_t LDS = (2 * TILE * BUFS + VALS) * 2 + BUFS * 2 * BR * 4;
};

template <int TY, int DP>
__global__ __launch_bounds__(256, (DkvCfg<TY, DP>::WAVES)) void bwd_dkv_kernel(const Args a) {
    using C = DkvCfg<TY, DP>;
    using T = Ty<TY>;
    extern __shared__ __attribute__((aligned(16))) short lds[];
    short* const vals = lds + 2 * C::TILE * C::BUFS;
    float* const stat = reinterpret_cast<float*>(vals + C::VALS);          // [BUFS][BR log-sums, BR negative deltas] of the tile's rows
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int rest = uniform(id / a.tiles), tile = id - rest * a.tiles, bh = uniform(rest / a.nsplit), split = rest - bh * a.nsplit;
    const int b = uniform(bh / a.Hkv), kv = bh - b * a.Hkv;
    const int key = tile * C::KEYS + 32 * w + (lane & 31);
    const bool in = key < a.Lk, live = in && !(a.pad && a.pad[b * a.pad_b + key]);
    const bool work = __builtin_amdgcn_ballot_w64(live) != 0;             // of this wave
    const int r0 = split * a.span, rend = __builtin_amdgcn_readfirstlane(__syncthreads_or(work)) ? min(a.R, r0 + a.span) : r0;

    Stage<TY, DP, C::BR, C::NT> sq, sd;
    float st = 0.f;
    const char* const qb = (const char*)a.q + (b * a.q_b + (int64_t)kv * a.G * a.q_h) * T::ES;
    const char* const db = (const char*)a.dout + (b * a.d_b + (int64_t)kv * a.G * a.d_h) * T::ES;
    const auto fetch = [&](int r) {
        const int g0 = uniform(r / a.Lq), i0 = r - g0 * a.Lq, here = min(rend - r, a.Lq - i0);      // rows of head g0 from here on
        if (here >= C::BR) {                                               // the tile's rows are of one head
            sq.load(tid, a.D, qb + (i0 * a.q_l + g0 * a.q_h) * T::ES, a.q_l * T::ES, here);
            sd.load(tid, a.D, db + (i0 * a.d_l + g0 * a.d_h) * T::ES, a.d_l * T::ES, here);
        } else {
            // Behind the last row: its query again, whose score with an infinite key is no NaN unless that row's own is (zeros would make one),
            // and an output gradient of zeros; the log-sum of +infinity makes its probabilities 0.
            const auto at = [&](int x, const char* base, int64_t sl, int64_t sh) {
                const int g = x / a.Lq, i = x - g * a.Lq;
                return base + (i * sl + g * sh) * T::ES;
            };
            sq.gather(tid, a.D, [&](int x) { return at(min(r + x, rend - 1), qb, a.q_l, a.q_h); });
            sd.gather(tid, a.D, [&](int x) { return r + x < rend ? at(r + x, db, a.d_l, a.d_h) : nullptr; });
        }
        const int x = r + tid % C::BR;
        if (tid < C::BR) st = x < rend ? a.lse[(int64_t)bh * a.R + x] - T::PSHIFT : INFINITY;
        else if (tid < 2 * C::BR) st = x < rend ? -a.delta[(int64_t)bh * a.R + x] : 0.f;
    };
    if (r0 < rend) fetch(r0);

    Frag<T::PL> kf[DP / 16], vf[C::VALS ? 1 : DP / 16];
    load_row<TY, DP>(live ? (const char*)a.k + (b * a.k_b + key * a.k_l + kv * a.k_h) * T::ES : nullptr, a.D, lane, kf);
    if constexpr (C::VALS == 0) {
        load_row<TY, DP>(live ? (const char*)a.v + (b * a.v_b + key * a.v_l + kv * a.v_h) * T::ES : nullptr, a.D, lane, vf);
    } else if (r0 < rend) {
        const int k0 = tile * C::KEYS, left = a.Lk - k0;
        const uint8_t* const pad = a.pad ? a.pad + b * a.pad_b + k0 : nullptr;
        Stage<TY, DP, C::KEYS, C::NT> sv;
        sv.load(tid, a.D, (const char*)a.v + (b * a.v_b + k0 * a.v_l + kv * a.v_h) * T::ES, a.v_l * T::ES, left);
        if (pad) {
            const unsigned long long w0 = __builtin_amdgcn_ballot_w64(lane < left && !pad[lane]);
            const unsigned long long w1 = __builtin_amdgcn_ballot_w64(64 + lane < left && !pad[64 + lane]);
            sv.blank(tid, [&](int r) { return (bool)((r >= 64 ? w1 >> (r & 63) : w0 >> (r & 63)) & 1ull); });
        }
        sv.store(vals, tid);                                               // the loop's barrier stands between this and the first read
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dk[t] = dv[t] = zero16();
    DsScale<TY, DP / 32> sc;

    int buf = 0;
    for (int r = r0; r < rend; r += C::BR) {
        short* const qt = lds + buf * 2 * C::TILE;
        short* const dt = qt + C::TILE;
        float* const lsd = stat + buf * 2 * C::BR;
        if (C::BUFS == 1) __syncthreads();
        sq.store(qt, tid);
        sd.store(dt, tid);
        if (tid < 2 * C::BR) lsd[tid] = st;
        __syncthreads();
        if (r + C::BR < rend) fetch(r + C::BR);
        if (C::BUFS == 2) buf ^= 1;
        if (!work) continue;
#pragma unroll
        for (int t = 0; t < C::BR / 32; ++t) {
            f32x16 s = zero16(), dp;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) s = mma<TY>(row_frag<TY, DP, C::BR>(qt, 32 * t, 16 * d, lane), kf[d], s);
            const auto products = [&] {
                dp = start16(lsd + C::BR + 32 * t, half);                  // dp - delta: the sums start at -delta
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    if constexpr (C::VALS == 0) dp = mma<TY>(row_frag<TY, DP, C::BR>(dt, 32 * t, 16 * d, lane), vf[d], dp);
                    else dp = mma<TY>(row_frag<TY, DP, C::BR>(dt, 32 * t, 16 * d, lane), row_frag<TY, DP, C::KEYS>(vals, 32 * w, 16 * d, lane), dp);
                }
            };
            if constexpr (!C::TIGHT) products();                            // beside the exponentials; registers have no room for both above
            else __builtin_amdgcn_sched_barrier(0);
            float p[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const fx4 ls = *reinterpret_cast<const fx4*>(lsd + 32 * t + 8 * g + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[4 * g + i] = exp2_f(fmaf(s[4 * g + i], a.c, -ls[i]));
            }
            {
                const Frag<T::PL> p0 = make_frag<TY, true>(p), p1 = make_frag<TY, true>(p + 8);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    dv[d] = mma<TY>(col_frag<TY, DP, C::BR>(dt, 32 * t, 32 * d, lane), p0, dv[d]);
                    dv[d] = mma<TY>(col_frag<TY, DP, C::BR>(dt, 32 * t + 16, 32 * d, lane), p1, dv[d]);
                }
            }
            if constexpr (C::TIGHT) {
                __builtin_amdgcn_sched_barrier(0);
                products();
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] *= dp[i];
            sc.fit(p, dk);
            const Frag<T::PL> d0 = make_frag<TY>(p), d1 = make_frag<TY>(p + 8);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                dk[d] = mma<TY>(col_frag<TY, DP, C::BR>(qt, 32 * t, 32 * d, lane), d0, dk[d]);
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
// forward: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  Few splits: a thread owns four columns of a row, bound by the partial
// results' bytes (two splits of 32768 x 128 columns, 50 MB with the result: 10 us).
constexpr int MOST_SPLITS = 1024, FEW_SPLITS = 8;
constexpr float SPARE = 1.f / MOST_SPLITS;               // the weights are formed times this: their sum with values near the largest stays in range

template <int TY>
__global__ __launch_bounds__(256) void join_few_kernel(const Args a) {
    const int nq = a.D / 4;
    const int64_t rows = (int64_t)a.B * a.Hkv * a.R, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * nq) return;
    const int64_t fr = e / nq;
    const int d = 4 * (int)(e % nq);
    float ls[FEW_SPLITS], M = -INFINITY, W = 0.f;
    fx4 y[FEW_SPLITS], x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        ls[s] = -INFINITY;
        y[s] = x;
        if (s < a.nsplit) {
            ls[s] = a.part_lse[s * rows + fr];
            y[s] = *reinterpret_cast<const fx4*>(a.part + (s * rows + fr) * a.D + d);
        }
        M = fmaxf(M, ls[s]);
    }
    const float mr = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        const float wgt = exp2_f(ls[s] - mr) * SPARE;
        W += wgt;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(wgt, y[s][j], x[j]);
    }
    const float inv = W == 0.f ? 0.f : M == NO_SCORE ? no_sum(true) : 1.f / W;
    const int64_t at = out_at(a, (int)(fr / a.R), (int)(fr % a.R)) + d;
    put4<TY>(a.o, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (a.o32) put4<F32>(a.o32, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (d == 0 && a.lse) a.lse[fr] = W == 0.f ? INFINITY : M == NO_SCORE ? no_lse(true) : M + __builtin_amdgcn_logf(W * (1.f / SPARE));
}

// Many splits: a workgroup owns a row, its threads take four columns of every (256 / columns)-th split, so that one latency covers many
// splits, and are summed in a fixed order.  128 rows of 16 splits of 128 columns: 5 us, a launch and two latencies.
template <int TY>
__global__ __launch_bounds__(256) void join_fwd_kernel(const Args a) {
    __shared__ float wgt[MOST_SPLITS], part[256][4], red[8];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t rows = (int64_t)a.B * a.Hkv * a.R, fr = blockIdx.x;
    float M = -INFINITY;
    for (int s = tid; s < a.nsplit; s += 256) M = fmaxf(M, wgt[s] = a.part_lse[s * rows + fr]);
    M = wave_max(M);
    if (lane == 0) red[w] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mr = M == -INFINITY ? 0.f : M;
    float W = 0.f;
    for (int s = tid; s < a.nsplit; s += 256) W += wgt[s] = exp2_f(wgt[s] - mr) * SPARE;
    W = wave_sum(W);
    if (lane == 0) red[4 + w] = W;
    __syncthreads();
    W = red[4] + red[5] + red[6] + red[7];
    const float inv = W == 0.f ? 0.f : M == NO_SCORE ? no_sum(true) : 1.f / W;
    const int nq = a.D / 4, ng = 256 / nq, g = tid / nq, d = 4 * (tid % nq);
    fx4 x = {0.f, 0.f, 0.f, 0.f};
    if (g < ng)
        for (int s = g; s < a.nsplit; s += ng) {
            const fx4 y = *reinterpret_cast<const fx4*>(a.part + (s * rows + fr) * a.D + d);
            const float f = wgt[s];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fmaf(f, y[j], x[j]);
        }
    *reinterpret_cast<fx4*>(part[tid]) = x;
    __syncthreads();
    if (g) return;
    for (int i = 1; i < ng; ++i) {
        const fx4 y = *reinterpret_cast<const fx4*>(part[i * nq + tid]);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += y[j];
    }
    const int bh = (int)(fr / a.R), r = (int)(fr % a.R);
    const int64_t at = out_at(a, bh, r) + d;
    put4<TY>(a.o, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (a.o32) put4<F32>(a.o32, at, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (d == 0 && a.lse) a.lse[fr] = W == 0.f ? INFINITY : M == NO_SCORE ? no_lse(true) : M + __builtin_amdgcn_logf(W * (1.f / SPARE));
}
// backward: out[i] = sum_s part[s][i], s ascending; n a multiple of 4.  8 splits of 0.5 M values: 5 us, about half of it the launch.  Sixteen
// loads in flight: a small output has few threads, and one load at a time cost a memory latency a split (683 splits of 512 values: 172 us).
template <int COUNT>
__device__ __forceinline__ void add_splits(fx4& x, const float* part, int64_t n) {
    fx4 y[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) y[i] = *reinterpret_cast<const fx4*>(part + i * n);
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += y[i][j];
}
template <int TY>
__global__ __launch_bounds__(256) void join_sum_kernel(const float* part, void* out, int64_t n, int nsplit) {
    const int64_t e = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (e >= n) return;
    fx4 x = *reinterpret_cast<const fx4*>(part + e);
    int s = 1;
    for (; s + 16 <= nsplit; s += 16) add_splits<16>(x, part + s * n + e, n);
    for (; s + 4 <= nsplit; s += 4) add_splits<4>(x, part + s * n + e, n);
    for (; s < nsplit; ++s) add_splits<1>(x, part + s * n + e, n);
    put4<TY>(out, e, x[0], x[1], x[2], x[3]);
}

// ---- launches of one element type (defined in that type's unit) -------------------------------------------------------------------------
template <int TY> int launch_fwd(const Args& a, int few, hipStream_t s);
template <int TY> int launch_join_fwd(const Args& a, hipStream_t s);
template <int TY> int launch_bwd_dq(const Args& a, hipStream_t s);
template <int TY> int launch_bwd_dkv(const Args& a, hipStream_t s);
template <int TY> int launch_join_sum(const float* part, void* out, int64_t n, int nsplit, hipStream_t s);

}  // namespace xattn
