// Token embedding: rows of a table by given ids, times a factor, and the table's gradient by sorted tokens.
//   out[t] = scale * W[ids[t]]                               dW[v] = scale * sum of dout[t] over ids[t] == v (t ascending)
// Both are memory-bound: the forward pass is one gather; the gradient reads every row of dout once and writes every row of dW.
// The gradient has no float atomics: a stable radix sort brings equal ids together (integer counts only, so its order is fixed), each
// wave sums a run of sorted positions in fp32 registers, runs that cross a chunk's border are joined in chunk order by a last pass.
#include "common.h"

namespace {

typedef __bf16 eb2 __attribute__((ext_vector_type(2)));
typedef _Float16 eh2 __attribute__((ext_vector_type(2)));
typedef float ef2 __attribute__((ext_vector_type(2)));
enum { F32 = 0, BF16 = 1, F16 = 2 };

template <int TY> __device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (TY == F16) return __builtin_bit_cast(unsigned, __builtin_convertvector((ef2){a, b}, eh2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector((ef2){a, b}, eb2));
}
template <int TY> __device__ __forceinline__ ef2 unpack2(unsigned u) {
    if constexpr (TY == F16) return __builtin_convertvector(__builtin_bit_cast(eh2, u), ef2);
    else return (ef2){__builtin_bit_cast(float, u << 16), __builtin_bit_cast(float, u & 0xffff0000u)};
}
// one lane's share of a row: a 16-byte chunk (VEC) or one element
template <int TY, bool VEC> struct Piece {
    static constexpr int ES = TY == F32 ? 4 : 2;
    static constexpr int N = VEC ? 16 / ES : 1;
    float x[N];
    __device__ __forceinline__ void load(const void* p, int64_t e) {
        if constexpr (VEC) {
            const u32x4_t u = *reinterpret_cast<const u32x4_t*>((const char*)p + e * ES);
            if constexpr (TY == F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { const unsigned e = u[i]; x[i] = __builtin_bit_cast(float, e); }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) { const ef2 w = unpack2<TY>(u[i]); x[2 * i] = w.x; x[2 * i + 1] = w.y; }
            }
        } else if constexpr (TY == F32) {
            x[0] = ((const float*)p)[e];
        } else {
            x[0] = unpack2<TY>(((const unsigned short*)p)[e]).x;
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t e) const {
        if constexpr (VEC) {
            u32x4_t u;
            if constexpr (TY == F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(unsigned, x[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = pack2<TY>(x[2 * i], x[2 * i + 1]);
            }
            *reinterpret_cast<u32x4_t*>((char*)p + e * ES) = u;
        } else if constexpr (TY == F32) {
            ((float*)p)[e] = x[0];
        } else {
            ((unsigned short*)p)[e] = (unsigned short)pack2<TY>(x[0], 0.f);
        }
    }
};

template <typename I> __device__ __forceinline__ int64_t id_at(const void* ids, int64_t t) { return (int64_t)((const I*)ids)[t]; }

// A block takes `rows` tokens of `cpr` pieces each; four pieces of a thread are in flight.  An id outside [0, V) reads nothing and gives
// NaN.  At 65536 x 1024 fp16 the launch moves 268 MB.
template <int TY, bool VEC, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* ids, const void* w, int64_t w_stride, int64_t V, void* out, int64_t T,
                                                        int C, int cpr, int rows, float scale) {
    using P = Piece<TY, VEC>;
    const int64_t t0 = (int64_t)blockIdx.x * rows;
    const int n = (int)(T - t0 < rows ? T - t0 : rows) * cpr;
    for (int e0 = threadIdx.x; e0 < n; e0 += 1024) {
        P p[4];
        int64_t to[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = e0 + 256 * u;
            to[u] = -1;
            if (e < n) {
                const int r = e / cpr, c = (e - r * cpr) * P::N;
                const int64_t id = id_at<I>(ids, t0 + r);
                to[u] = (t0 + r) * C + c;
                if (id >= 0 && id < V) {
                    p[u].load(w, id * w_stride + c);
                } else {
#pragma unroll
                    for (int i = 0; i < P::N; ++i) p[u].x[i] = __builtin_nanf("");
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (to[u] >= 0) {
#pragma unroll
                for (int i = 0; i < P::N; ++i) p[u].x[i] *= scale;
                p[u].store(out, to[u]);
            }
    }
}

// ---- stable sort of (id, t) by id: 8 bits a pass, least significant first -----------------------------------------------------------
// Block b owns `tpb` consecutive entries.  count[p][digit][block]: how many entries of the block have that digit of pass p.  The counts
// of pass 0 are written by embed_count_kernel, those of a later pass by atomic adds of the pass before it (an entry knows where it goes;
// integer counts do not depend on the order).  Ids outside [0, V) and the padding id are left out; *valid = entries that remain.
constexpr int DIGITS = 256, SORT_BLOCKS = 256, BATCH = 1024;

template <typename I>
__device__ __forceinline__ bool entry_of(const void* ids, int64_t t, int64_t V, int64_t padding, unsigned& key) {
    const int64_t id = id_at<I>(ids, t);
    key = (unsigned)id;
    return id >= 0 && id < V && id != padding;
}

// counts of pass 0, zeros for the later passes' counts and for the whole gradient (rows that no token names keep them)
template <typename I>
__global__ __launch_bounds__(256) void embed_count_kernel(const void* ids, int64_t T, int64_t V, int64_t padding, int tpb, int nblk, int passes,
                                                          unsigned* count, void* dw, int64_t dw_bytes) {
    __shared__ unsigned h[DIGITS];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < nblk) {
        h[tid] = 0;
        __syncthreads();
        const int64_t t0 = (int64_t)blockIdx.x * tpb, t1 = t0 + tpb < T ? t0 + tpb : T;
        for (int64_t t = t0 + tid; t < t1; t += 256) {
            unsigned key;
            if (entry_of<I>(ids, t, V, padding, key)) atomicAdd(&h[key & 255u], 1u);
        }
        __syncthreads();
        count[tid * nblk + blockIdx.x] = h[tid];
        for (int p = 1; p < passes; ++p) count[(p * DIGITS + tid) * nblk + blockIdx.x] = 0;
    }
    const int64_t n16 = dw_bytes / 16, step = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + tid;
    const u32x4_t z = {0u, 0u, 0u, 0u};
    for (int64_t i = i0; i < n16; i += step) reinterpret_cast<u32x4_t*>(dw)[i] = z;
    if (i0 < dw_bytes % 16) ((char*)dw)[n16 * 16 + i0] = 0;
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const void* ids, const uint2* in, uint2* out, int64_t T, int64_t V, int64_t padding,
                                                            int tpb, int nblk, int pass, int passes, unsigned* count, unsigned* valid) {
    __shared__ unsigned run[DIGITS], wcount[4][DIGITS], wsum[4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, blk = blockIdx.x;
    // where this block's entries of digit `tid` begin: all smaller digits, and the same digit of the blocks before
    unsigned before = 0, total = 0;
    const unsigned* c = count + ((int64_t)pass * DIGITS + tid) * nblk;
    for (int i = 0; i < nblk; ++i) {
        const unsigned x = c[i];
        before += i < blk ? x : 0;
        total += x;
    }
    unsigned inc = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned y = __shfl_up(inc, o, 64);
        if (lane >= o) inc += y;
    }
    if (lane == 63) wsum[w] = inc;
    __syncthreads();
    unsigned base = inc - total;
    for (int i = 0; i < w; ++i) base += wsum[i];
    run[tid] = base + before;
    if (blk == 0 && tid == 255) *valid = base + total;
    const int64_t n = FIRST ? T : (int64_t)(wsum[0] + wsum[1] + wsum[2] + wsum[3]);
    const int64_t t0 = (int64_t)blk * tpb, t1 = t0 + tpb < n ? t0 + tpb : n;

    for (int64_t b0 = t0; b0 < t1; b0 += BATCH) {                          // a wave owns 256 consecutive entries of the batch
        unsigned key[4], idx[4];
        bool live[4];
        __syncthreads();                                                   // run[] is final, wcount[] free
#pragma unroll
        for (int i = 0; i < 4; ++i) wcount[i][tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t t = b0 + 256 * w + 64 * i + lane;
            live[i] = t < t1;
            key[i] = idx[i] = 0;
            if (live[i]) {
                if constexpr (FIRST) {
                    live[i] = entry_of<I>(ids, t, V, padding, key[i]);
                    idx[i] = (unsigned)t;
                } else {
                    const uint2 e = in[t];
                    key[i] = e.x; idx[i] = e.y;
                }
            }
            if (live[i]) atomicAdd(&wcount[w][key[i] >> (8 * pass) & 255u], 1u);
        }
        __syncthreads();
        {
            unsigned at = run[tid];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned x = wcount[i][tid];
                wcount[i][tid] = at;
                at += x;
            }
            run[tid] = at;
        }
        __syncthreads();
        volatile unsigned* const place = wcount[w];                        // this wave's next free place of every digit
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned dig = key[i] >> (8 * pass) & 255u;
            unsigned long long same = __builtin_amdgcn_ballot_w64(live[i]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool bit = dig >> k & 1u;
                const unsigned long long v = __builtin_amdgcn_ballot_w64(bit);
                same &= bit ? v : ~v;
            }
            const unsigned rank = __popcll(same & ((1ull << lane) - 1ull)), all = __popcll(same);
            unsigned to = 0;
            if (live[i]) to = place[dig] + rank;
            __builtin_amdgcn_wave_barrier();
            if (live[i] && rank == 0) place[dig] = to + all;
            __builtin_amdgcn_wave_barrier();
            if (live[i]) {
                out[to] = make_uint2(key[i], idx[i]);
                if (pass + 1 < passes)
                    atomicAdd(&count[((int64_t)(pass + 1) * DIGITS + (key[i] >> (8 * pass + 8) & 255u)) * nblk + to / (unsigned)tpb], 1u);
            }
        }
    }
}

// ---- sums of runs of equal ids --------------------------------------------------------------------------------------------------------
// A wave takes `chunk` sorted positions and 64 pieces of columns.  A run inside the chunk goes straight to dW; the part of a run that
// continues from the chunk before goes to part[c][0], the part of one that starts here and goes on to part[c][1].
template <int TY, bool VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const uint2* sorted, const unsigned* valid, const void* dout, void* dw, float* part,
                                                        int C, int chunk, int nseg, float scale) {
    using P = Piece<TY, VEC>;
    const int lane = threadIdx.x & 63;
    const int64_t n = *valid, u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t c = u / nseg, p0 = c * chunk, p1 = p0 + chunk < n ? p0 + chunk : n;
    const int col = ((int)(u - c * nseg) * 64 + lane) * P::N;
    if (p0 >= p1) return;
    const bool in = col < C;
    bool head = p0 > 0 && sorted[p0 - 1].x == sorted[p0].x;                // the first run came from the chunk before
    float acc[P::N];
#pragma unroll
    for (int i = 0; i < P::N; ++i) acc[i] = 0.f;
    constexpr int AHEAD = 8;
    for (int64_t q = p0; q < p1; q += AHEAD) {
        uint2 e[AHEAD + 1];
        P x[AHEAD];
#pragma unroll
        for (int i = 0; i <= AHEAD; ++i) {
            e[i] = make_uint2(0xffffffffu, 0u);                            // no id: ids are below 2^31
            if (q + i < n) e[i] = sorted[q + i];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (q + i < p1 && in) x[i].load(dout, (int64_t)e[i].y * C + col);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (q + i >= p1) break;
            if (in) {
#pragma unroll
                for (int j = 0; j < P::N; ++j) acc[j] += x[i].x[j];
            }
            const bool ends = e[i].x != e[i + 1].x, last = q + i + 1 == p1;
            if (!ends && !last) continue;
            if (in) {
                if (ends && !head) {
                    P r;
#pragma unroll
                    for (int j = 0; j < P::N; ++j) r.x[j] = acc[j] * scale;
                    r.store(dw, (int64_t)e[i].x * C + col);
                } else {
                    float* to = part + (2 * c + (head ? 0 : 1)) * C + col;
#pragma unroll
                    for (int j = 0; j < P::N; ++j) to[j] = acc[j];
                }
            }
#pragma unroll
            for (int j = 0; j < P::N; ++j) acc[j] = 0.f;
            head = false;
        }
    }
}

// A run that starts in chunk c and goes on: its part there and those of the chunks that follow, in order
template <int TY, bool VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(const uint2* sorted, const unsigned* valid, void* dw, const float* part, int C,
                                                         int chunk, int nseg, float scale) {
    using P = Piece<TY, VEC>;
    const int lane = threadIdx.x & 63;
    const int64_t n = *valid, u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t c = u / nseg, p0 = c * chunk, p1 = p0 + chunk;
    const int col = ((int)(u - c * nseg) * 64 + lane) * P::N;
    if (p1 >= n) return;                                                   // the last chunk's runs end in it
    const unsigned id = sorted[p1 - 1].x;
    if (sorted[p1].x != id) return;
    if (sorted[p0].x == id && p0 > 0 && sorted[p0 - 1].x == id) return;    // it started before this chunk
    int64_t end = c + 1;                                                   // last chunk that holds a part of the run
    {
        int64_t lo = c + 1, hi = (n - 1) / chunk;                          // first position of chunk lo has the id
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) / 2;
            if (sorted[mid * chunk].x == id) lo = mid;
            else hi = mid - 1;
        }
        end = lo;
    }
    if (col >= C) return;
    P acc;
#pragma unroll
    for (int j = 0; j < P::N; ++j) acc.x[j] = part[(2 * c + 1) * C + col + j];
    constexpr int AHEAD = 8;
    for (int64_t k = c + 1; k <= end; k += AHEAD) {
        float x[AHEAD][P::N];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < P::N; ++j) x[i][j] = k + i <= end ? part[2 * (k + i) * C + col + j] : 0.f;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < P::N; ++j) acc.x[j] += x[i][j];
    }
#pragma unroll
    for (int j = 0; j < P::N; ++j) acc.x[j] *= scale;
    acc.store(dw, (int64_t)id * C + col);
}

struct Plan {
    int tpb, nblk, passes, chunk;
    int64_t chunks;
    size_t pairs, counts, parts, total;                                    // byte offsets of the workspace behind the first pair buffer
};
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

Plan plan(int64_t T, int64_t V, int C) {
    Plan p{};
    int64_t tpb = (T + SORT_BLOCKS - 1) / SORT_BLOCKS;
    tpb = (tpb + BATCH - 1) / BATCH * BATCH;
    p.tpb = (int)tpb;
    p.nblk = (int)((T + tpb - 1) / tpb);
    p.passes = 1;
    while (p.passes < 4 && (V - 1) >> (8 * p.passes)) ++p.passes;
    int64_t chunk = T / 4096 / 8 * 8;                                      // at most about 4096 chunks: a run that fills them all is joined by one wave
    p.chunk = (int)(chunk < 32 ? 32 : chunk);
    p.chunks = (T + p.chunk - 1) / p.chunk;
    p.pairs = up16((size_t)T * 8);
    p.counts = 2 * p.pairs;
    p.parts = p.counts + up16(((size_t)p.passes * DIGITS * p.nblk + 4) * 4);
    p.total = p.parts + (size_t)p.chunks * 2 * C * 4;
    return p;
}

bool vec_ok(int ty, int C, int64_t stride, const void* a, const void* b) {
    const int n = ty == F32 ? 4 : 8;
    return C % n == 0 && stride % n == 0 && ((((uintptr_t)a) | ((uintptr_t)b)) & 15) == 0;
}

template <int TY, bool VEC>
int go_fwd(const void* ids, int i64, const void* w, int64_t ws, int64_t V, void* out, int64_t T, int C, float scale, hipStream_t s) {
    const int cpr = C / Piece<TY, VEC>::N;
    const int rows = cpr >= 1024 ? 1 : 1024 / cpr;
    const int64_t blocks = (T + rows - 1) / rows;
    if (blocks > 0x7fffffff) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    if (i64) FAVAE_KLAUNCH((embed_fwd_kernel<TY, VEC, int64_t>), dim3((unsigned)blocks), dim3(256), 0, s, ids, w, ws, V, out, T, C, cpr, rows, scale);
    else FAVAE_KLAUNCH((embed_fwd_kernel<TY, VEC, int32_t>), dim3((unsigned)blocks), dim3(256), 0, s, ids, w, ws, V, out, T, C, cpr, rows, scale);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}

template <int TY, bool VEC>
int go_sums(const uint2* sorted, const unsigned* valid, const void* dout, void* dw, float* part, int C, const Plan& p, float scale, hipStream_t s) {
    const int per = 64 * Piece<TY, VEC>::N, nseg = (C + per - 1) / per;
    const int64_t blocks = (p.chunks * nseg + 3) / 4;
    if (blocks > 0x7fffffff) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    FAVAE_KLAUNCH((embed_sum_kernel<TY, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, sorted, valid, dout, dw, part, C, p.chunk, nseg, scale);
    FAVAE_CHECK_LAUNCH();
    if (p.chunks > 1) {
        FAVAE_KLAUNCH((embed_join_kernel<TY, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, sorted, valid, dw, (const float*)part, C, p.chunk, nseg, scale);
        FAVAE_CHECK_LAUNCH();
    }
    return FAVAE_OK;
}

bool ok_sizes(int64_t T, int64_t V, int C, int ty) {
    return T >= 1 && T < ((int64_t)1 << 31) - 1 && V >= 1 && V < ((int64_t)1 << 31) && C >= 1 && C <= (1 << 24) && ty >= F32 && ty <= F16;
}

}  // namespace

extern "C" int favae_embed_fwd(const void* ids, int ids_are_64bit, const void* weight, int64_t weight_stride, int64_t V, void* out, int64_t T,
                               int C, int dtype, float scale, favae_stream_t stream) {
    FAVAE_REQUIRE(ids && weight && out && weight_stride >= 0);
    if (!ok_sizes(T, V, C, dtype)) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    const hipStream_t s = (hipStream_t)stream;
    const bool vec = vec_ok(dtype, C, weight_stride, weight, out);
#define GO(TY)                                                                                                            \
    return vec ? go_fwd<TY, true>(ids, ids_are_64bit, weight, weight_stride, V, out, T, C, scale, s)                      \
               : go_fwd<TY, false>(ids, ids_are_64bit, weight, weight_stride, V, out, T, C, scale, s)
    if (dtype == F32) GO(F32);
    if (dtype == BF16) GO(BF16);
    GO(F16);
#undef GO
}

extern "C" size_t favae_embed_bwd_workspace(int64_t T, int64_t V, int C) {
    return ok_sizes(T, V, C, F32) ? plan(T, V, C).total : 0;
}

extern "C" int favae_embed_bwd(const void* ids, int ids_are_64bit, const void* dout, int64_t T, int64_t V, int C, int dtype, float scale,
                               int64_t padding_idx, void* dweight, void* ws, size_t ws_bytes, favae_stream_t stream) {
    FAVAE_REQUIRE(ids && dout && dweight && ws);
    if (!ok_sizes(T, V, C, dtype) || ((uintptr_t)ws & 15) || ((uintptr_t)dweight & 15)) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    const Plan p = plan(T, V, C);
    if (ws_bytes < p.total) return favae_prof_fail_(FAVAE_ERR_WORKSPACE);
    const hipStream_t s = (hipStream_t)stream;
    uint2* const buf[2] = {(uint2*)ws, (uint2*)((char*)ws + p.pairs)};
    unsigned* const count = (unsigned*)((char*)ws + p.counts);
    unsigned* const valid = count + (size_t)p.passes * DIGITS * p.nblk;
    float* const part = (float*)((char*)ws + p.parts);
    const int64_t dw_bytes = V * C * (dtype == F32 ? 4 : 2);
    const int64_t zb = (dw_bytes + 65535) / 65536;
    const int grid = (int)(zb > 2048 ? 2048 : zb > p.nblk ? zb : p.nblk);
    if (ids_are_64bit) FAVAE_KLAUNCH((embed_count_kernel<int64_t>), dim3(grid), dim3(256), 0, s, ids, T, V, padding_idx, p.tpb, p.nblk, p.passes, count, dweight, dw_bytes);
    else FAVAE_KLAUNCH((embed_count_kernel<int32_t>), dim3(grid), dim3(256), 0, s, ids, T, V, padding_idx, p.tpb, p.nblk, p.passes, count, dweight, dw_bytes);
    FAVAE_CHECK_LAUNCH();
    for (int k = 0; k < p.passes; ++k) {
        const uint2* in = buf[(k + 1) & 1];
        uint2* out = buf[k & 1];
        if (k) FAVAE_KLAUNCH((embed_scatter_kernel<int32_t, false>), dim3(p.nblk), dim3(256), 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, p.passes, count, valid);
        else if (ids_are_64bit) FAVAE_KLAUNCH((embed_scatter_kernel<int64_t, true>), dim3(p.nblk), dim3(256), 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, p.passes, count, valid);
        else FAVAE_KLAUNCH((embed_scatter_kernel<int32_t, true>), dim3(p.nblk), dim3(256), 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, p.passes, count, valid);
        FAVAE_CHECK_LAUNCH();
    }
    const uint2* sorted = buf[(p.passes - 1) & 1];
    const bool vec = vec_ok(dtype, C, 0, dout, dweight);
#define GO(TY)                                                                                      \
    return vec ? go_sums<TY, true>(sorted, valid, dout, dweight, part, C, p, scale, s)              \
               : go_sums<TY, false>(sorted, valid, dout, dweight, part, C, p, scale, s)
    if (dtype == F32) GO(F32);
    if (dtype == BF16) GO(BF16);
    GO(F16);
#undef GO
}
