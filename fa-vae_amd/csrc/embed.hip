// Token embedding: rows of a table by given ids, times a factor, and the table's gradient by sorted tokens.
//   out[t] = scale * W[ids[t]]                               dW[v] = scale * sum of dout[t] over ids[t] == v (t ascending)
// Both are memory-bound: the forward pass is one gather; the gradient reads every row of dout once and writes every row of dW.
// The gradient has no float atomics: a stable radix sort brings equal ids together (integer counts only, so its order is fixed), each
// wave sums a run of sorted positions in fp32 registers, runs that cross a chunk's border are joined in chunk order by a last pass.
// Sums are fp32 for every type; a result is rounded once.
// Measured (times of the kernels alone; 64 K tokens):
//   8192 x 256 fp32, uniform ids     forward 19 us, gradient 42: counts 5 + 4, scatters 7 + 7, sums 14 (5.3 TB/s), joins 4
//   49999 x 768 bf16, 1 / rank ids   forward 30 us, gradient 63: counts and zeros 12 + 4, scatters 7 + 7, sums 26 (4.4 TB/s), joins 11
// The four launches of the sort move under 3 MB: they are bound by launches and latencies, at least 3 us each.
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
// NaN.  Bound by the writes: 65536 tokens x 1024 fp16 out of 16384 rows (34 MB) are 168 MB in 29 us, 5.8 TB/s; one token 1.4 us.
template <int TY, bool VEC, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* ids, const void* w, int64_t w_stride, int64_t V, void* out, int64_t T,
                                                        int C, int cpr, int rows, float scale) {
    using P = Piece<TY, VEC>;
    const int64_t t0 = (int64_t)blockIdx.x * rows;
    const int n = (int)(T - t0 < rows ? T - t0 : rows) * cpr;
    for (int e0 = threadIdx.x; e0 < n; e0 += 1024) {
        P p[4];
        int64_t id[4];
        int r[4], c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {                                      // no branch: the four loads of each kind are in flight together
            const int e = min(e0 + 256 * u, n - 1);
            r[u] = e / cpr;
            c[u] = (e - r[u] * cpr) * P::N;
            id[u] = id_at<I>(ids, t0 + r[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u].load(w, (id[u] >= 0 && id[u] < V ? id[u] : 0) * w_stride + c[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (e0 + 256 * u < n) {
                const bool ok = id[u] >= 0 && id[u] < V;
#pragma unroll
                for (int i = 0; i < P::N; ++i) p[u].x[i] = ok ? p[u].x[i] * scale : __builtin_nanf("");
                p[u].store(out, (t0 + r[u]) * C + c[u]);
            }
    }
}

// ---- stable sort of (id, t) by id: 8 bits a pass, least significant first -----------------------------------------------------------
// Block b owns `tpb` consecutive entries.  count[digit][block]: how many entries of the block have that digit of this pass (integer
// counts, so nothing depends on the order of the LDS atomics).  Ids outside [0, V) and the padding id are left out; *valid = entries
// that remain.  Up to SMALL tokens are sorted by one workgroup in LDS in one launch.
constexpr int DIGITS = 256, SORT_BLOCKS = 256, BATCH = 1024, SMALL = 2048;
__host__ __device__ constexpr int up4(int n) { return (n + 3) & ~3; }      // a digit's counts begin at 16 bytes

template <typename I>
__device__ __forceinline__ bool entry_of(const void* ids, int64_t t, int64_t V, int64_t padding, unsigned& key) {
    const int64_t id = id_at<I>(ids, t);
    key = (unsigned)id;
    return id >= 0 && id < V && id != padding;
}

// zeros for the whole gradient (rows that no token names keep them): blocks [first, gridDim.x)
__device__ __forceinline__ void clear_rows(void* dw, int64_t bytes, int first) {
    const int64_t n16 = bytes / 16, step = (int64_t)(gridDim.x - first) * 256, i0 = (int64_t)(blockIdx.x - first) * 256 + threadIdx.x;
    const u32x4_t z = {0u, 0u, 0u, 0u};
    for (int64_t i = i0; i < n16; i += step) reinterpret_cast<u32x4_t*>(dw)[i] = z;
    if (i0 < bytes % 16) ((char*)dw)[n16 * 16 + i0] = 0;
}

// counts of one pass; the first one also clears the gradient
template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void embed_count_kernel(const void* ids, const uint2* in, int64_t T, int64_t V, int64_t padding, int tpb, int nblk,
                                                          int pass, unsigned* count, const unsigned* valid, void* dw, int64_t dw_bytes) {
    __shared__ unsigned h[DIGITS];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < nblk) {
        h[tid] = 0;
        __syncthreads();
        const int64_t n = FIRST ? T : (int64_t)*valid, t0 = (int64_t)blockIdx.x * tpb, t1 = t0 + tpb < n ? t0 + tpb : n;
        for (int64_t t = t0 + tid; t < t1; t += 256) {
            unsigned key;
            bool live = true;
            if constexpr (FIRST) live = entry_of<I>(ids, t, V, padding, key);
            else key = in[t].x;
            if (live) atomicAdd(&h[key >> (8 * pass) & 255u], 1u);
        }
        __syncthreads();
        count[tid * up4(nblk) + blockIdx.x] = h[tid];
    }
    if (FIRST) clear_rows(dw, dw_bytes, 0);
}

// One batch of BATCH entries (a wave owns 256 consecutive ones, four of a lane): places of equal digits ascend with the entry.  run[digit]
// = the next free place, on entry and on return.
struct Ranker {
    unsigned run[DIGITS], wcount[4][DIGITS];

    template <typename Put>
    __device__ __forceinline__ void batch(const unsigned (&key)[4], const unsigned (&idx)[4], const bool (&live)[4], int shift, Put put) {
        const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
        __syncthreads();                                                   // run[] is final, wcount[] free
#pragma unroll
        for (int i = 0; i < 4; ++i) wcount[i][tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (live[i]) atomicAdd(&wcount[w][key[i] >> shift & 255u], 1u);
        __syncthreads();
        unsigned at = run[tid];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned x = wcount[i][tid];
            wcount[i][tid] = at;
            at += x;
        }
        run[tid] = at;
        __syncthreads();
        volatile unsigned* const place = wcount[w];                        // this wave's next free place of every digit
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned dig = key[i] >> shift & 255u;
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
            if (live[i]) put(to, key[i], idx[i]);
        }
    }
    // exclusive sums over the digits of `total`, one digit a thread; *all = their sum
    __device__ __forceinline__ unsigned before(unsigned total, unsigned* all) {
        __shared__ unsigned wsum[4];
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        unsigned inc = total;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned y = __shfl_up(inc, o, 64);
            if (lane >= o) inc += y;
        }
        __syncthreads();
        if (lane == 63) wsum[w] = inc;
        __syncthreads();
        unsigned base = inc - total;
        for (int i = 0; i < w; ++i) base += wsum[i];
        *all = wsum[0] + wsum[1] + wsum[2] + wsum[3];
        return base;
    }
};

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const void* ids, const uint2* in, uint2* out, int64_t T, int64_t V, int64_t padding,
                                                            int tpb, int nblk, int pass, const unsigned* count, unsigned* valid) {
    __shared__ Ranker rk;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, blk = blockIdx.x;
    I id[4];
    uint2 e[4];
    const int64_t t0 = (int64_t)blk * tpb;
    const auto fetch = [&](int64_t b0) {                                   // a batch's entries; the first one's are on their way under the counts
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t t = b0 + 256 * w + 64 * k + lane, at = t < T ? t : T - 1;
            if constexpr (FIRST) id[k] = ((const I*)ids)[at];
            else e[k] = in[at];
        }
    };
    fetch(t0);
    // where this block's entries of digit `tid` begin: all smaller digits, and the same digit of the blocks before
    unsigned before = 0, total = 0;
    const u32x4_t* const c = reinterpret_cast<const u32x4_t*>(count + (int64_t)tid * up4(nblk));
    const int quads = up4(nblk) / 4;
    for (int i = 0; i < quads; i += 16) {                                  // sixteen loads in flight: 64 blocks, one latency
        u32x4_t x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = c[min(i + j, quads - 1)];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int of = 4 * (i + j) + k;                            // its block; behind the last one: anything
                const unsigned n = x[j][k];
                before += of < blk ? n : 0;
                total += of < nblk ? n : 0;
            }
    }
    unsigned all;
    rk.run[tid] = rk.before(total, &all) + before;
    if (FIRST && blk == 0 && tid == 0) *valid = all;
    const int64_t n = FIRST ? T : (int64_t)all, t1 = t0 + tpb < n ? t0 + tpb : n;
    for (int64_t b0 = t0; b0 < t1; b0 += BATCH) {
        if (b0 > t0) fetch(b0);
        unsigned key[4], idx[4];
        bool live[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t t = b0 + 256 * w + 64 * k + lane;
            live[k] = t < t1;
            if constexpr (FIRST) {
                live[k] = live[k] && (int64_t)id[k] >= 0 && (int64_t)id[k] < V && (int64_t)id[k] != padding;
                key[k] = (unsigned)id[k];
                idx[k] = (unsigned)t;
            } else {
                key[k] = e[k].x;
                idx[k] = e[k].y;
            }
        }
        rk.batch(key, idx, live, 8 * pass, [&](unsigned to, unsigned k, unsigned t) { out[to] = make_uint2(k, t); });
    }
}

// All passes of up to SMALL tokens in one workgroup; the others clear the gradient.
template <typename I>
__global__ __launch_bounds__(256) void embed_sort_small_kernel(const void* ids, uint2* out, int T, int64_t V, int64_t padding, int passes,
                                                               unsigned* valid, void* dw, int64_t dw_bytes) {
    __shared__ Ranker rk;
    __shared__ uint2 buf[2][SMALL];
    __shared__ unsigned h[DIGITS];
    if (blockIdx.x) {
        clear_rows(dw, dw_bytes, 1);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int n = T;
    for (int pass = 0; pass < passes; ++pass) {
        h[tid] = 0;
        __syncthreads();
        const auto entry = [&](int t, unsigned& key, unsigned& idx) {
            bool live = t < n;
            key = idx = 0;
            if (live) {
                if (pass == 0) {
                    live = entry_of<I>(ids, t, V, padding, key);
                    idx = (unsigned)t;
                } else {
                    const uint2 e = buf[(pass + 1) & 1][t];
                    key = e.x;
                    idx = e.y;
                }
            }
            return live;
        };
        for (int t = tid; t < n; t += 256) {
            unsigned key, idx;
            if (entry(t, key, idx)) atomicAdd(&h[key >> (8 * pass) & 255u], 1u);
        }
        __syncthreads();
        unsigned all;
        rk.run[tid] = rk.before(h[tid], &all);
        const bool last = pass + 1 == passes;
        for (int b0 = 0; b0 < n; b0 += BATCH) {
            unsigned key[4], idx[4];
            bool live[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) live[k] = entry(b0 + 256 * w + 64 * k + lane, key[k], idx[k]);
            rk.batch(key, idx, live, 8 * pass, [&](unsigned to, unsigned k, unsigned t) {
                if (last) out[to] = make_uint2(k, t);
                else buf[pass & 1][to] = make_uint2(k, t);
            });
        }
        n = (int)all;
        __syncthreads();
    }
    if (tid == 0) *valid = (unsigned)n;
}

// ---- sums of runs of equal ids --------------------------------------------------------------------------------------------------------
// A wave takes `chunk` sorted positions and 64 pieces of columns.  A run inside the chunk goes straight to dW; the part of a run that
// continues from the chunk before goes to part[c][0], the part of one that starts here and goes on to part[c][1].
constexpr int GROUP = 32;        // positions whose ids and tokens one load brings: lane i holds position i

template <int TY, bool VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const uint2* sorted, const unsigned* valid, const void* dout, void* dw, float* part,
                                                        int64_t T, int C, int chunk, int nseg, float scale) {
    using P = Piece<TY, VEC>;
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t c = u / nseg, p0 = c * chunk;
    const int col = ((int)(u - c * nseg) * 64 + lane) * P::N;
    if (p0 >= T) return;
    uint2 e = sorted[p0 + lane < T ? p0 + lane : T - 1];                   // behind *valid: anything, not used
    const unsigned prev = sorted[p0 > 0 ? p0 - 1 : 0].x;
    const int64_t n = *valid, p1 = p0 + chunk < n ? p0 + chunk : n;
    if (p0 >= p1) return;
    const bool in = col < C;
    bool head = p0 > 0 && prev == (unsigned)__builtin_amdgcn_readlane((int)e.x, 0);       // the first run came from the chunk before
    float acc[P::N];
#pragma unroll
    for (int i = 0; i < P::N; ++i) acc[i] = 0.f;
    constexpr int AHEAD = 8;
    for (int64_t q0 = p0; q0 < p1; q0 += GROUP) {
        if (q0 > p0) e = sorted[q0 + lane < T ? q0 + lane : T - 1];
        if (q0 + lane >= n) e = make_uint2(0xffffffffu, 0u);               // no id: they are below 2^31
        const int m = p1 - q0 < GROUP ? (int)(p1 - q0) : GROUP;
        for (int j0 = 0; j0 < m; j0 += AHEAD) {
            P x[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)                                // no branch: all in flight (behind the end: the last row again)
                x[i].load(dout, (int64_t)(unsigned)__builtin_amdgcn_readlane((int)e.y, j0 + i < m ? j0 + i : m - 1) * C + (in ? col : 0));
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (j0 + i >= m) break;
                if (in) {
#pragma unroll
                    for (int j = 0; j < P::N; ++j) acc[j] += x[i].x[j];
                }
                const unsigned id = (unsigned)__builtin_amdgcn_readlane((int)e.x, j0 + i);
                const bool ends = id != (unsigned)__builtin_amdgcn_readlane((int)e.x, j0 + i + 1), last = q0 + j0 + i + 1 == p1;
                if (!ends && !last) continue;
                if (in) {
                    if (ends && !head) {
                        P r;
#pragma unroll
                        for (int j = 0; j < P::N; ++j) r.x[j] = acc[j] * scale;
                        r.store(dw, (int64_t)id * C + col);
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
}

// A run that starts in chunk c and goes on: its part there, then those of the chunks that follow.  A wave takes one run and 64 pieces of
// columns; a run of more than LONG parts is summed by the four waves of its workgroup, a contiguous quarter each, added in order.
constexpr int LONG = 16, JOIN = 4;       // JOIN: waves of a workgroup

template <int TY, bool VEC>
__global__ __launch_bounds__(64 * JOIN) void embed_join_kernel(const uint2* sorted, const unsigned* valid, void* dw, const float* part, int64_t T, int C,
                                                         int chunk, int64_t chunks, int nseg, float scale) {
    using P = Piece<TY, VEC>;
    __shared__ float sums[JOIN][64 * P::N];
    __shared__ int64_t run_end[JOIN];
    __shared__ unsigned run_id[JOIN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t u0 = (int64_t)blockIdx.x * JOIN, u = u0 + w, c = u / nseg, p0 = c * chunk, p1 = p0 + chunk;
    // one load for the ids around this chunk's borders and one for the first ids of the next 64 chunks (entries behind *valid hold anything)
    const int64_t near = lane == 0 ? p1 - 1 : lane == 1 ? p1 : lane == 2 ? p0 : p0 - 1, next = (c + 1 + lane) * chunk;
    const unsigned e = c < chunks && near >= 0 && near < T ? sorted[near].x : 0u, f = next < T ? sorted[next].x : 0u;
    const int64_t n = *valid, most = (n - 1) / chunk;
    const unsigned id = (unsigned)__builtin_amdgcn_readlane((int)e, 0);
    const bool goes_on = c < chunks && p1 < n && (unsigned)__builtin_amdgcn_readlane((int)e, 1) == id;
    const bool came = (unsigned)__builtin_amdgcn_readlane((int)e, 2) == id && p0 > 0 && (unsigned)__builtin_amdgcn_readlane((int)e, 3) == id;
    int64_t end = -1;                                                      // last chunk that holds a part of the run that starts here
    if (goes_on && !came) {
        end = c + __builtin_ctzll(~__builtin_amdgcn_ballot_w64(c + 1 + lane <= most && f == id) | 1ull << 63);
        if (end == c + 63) {                                               // all of them: the last one by sixty-fourths of what follows
            int64_t stop = most + 1;                                       // it is in [end, stop)
            while (stop - end > 1) {
                const int64_t step = (stop - end + 62) / 64, k = end + (lane + 1) * step;
                const unsigned long long has = __builtin_amdgcn_ballot_w64(k < stop && sorted[(k < stop ? k : end) * chunk].x == id);
                const int run = has == ~0ull ? 64 : __builtin_ctzll(~has);
                stop = stop < end + (run + 1) * step ? stop : end + (run + 1) * step;
                end += run * step;
            }
        }
    }
    const int seg = (int)(u - c * nseg);
    const auto total = [&](int64_t cc, int64_t k0, int64_t k1, bool with_start, int col, float (&acc)[P::N]) {
#pragma unroll
        for (int j = 0; j < P::N; ++j) acc[j] = with_start ? part[(2 * cc + 1) * C + (col < C ? col : 0) + j] : 0.f;
        constexpr int AHEAD = 8;
        for (int64_t k = k0; k <= k1; k += AHEAD) {
            // no branch: all in flight; those behind k1 are out of the buffer's range, which reads zeros and moves nothing
            const auto rs = make_rsrc(part + 2 * k * C, 0x7fffffffu);
            float x[AHEAD][P::N];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const unsigned at = k + i <= k1 && col < C ? 4u * (2u * i * (unsigned)C + (unsigned)col) : FAVAE_OOB;
                if constexpr (VEC) {
#pragma unroll
                    for (int j = 0; j < P::N; j += 4) {
                        const u32x4_t u = __builtin_amdgcn_raw_buffer_load_b128(rs, at + 4u * j, 0, 0);
#pragma unroll
                        for (int q = 0; q < 4; ++q) { const unsigned e = u[q]; x[i][j + q] = __builtin_bit_cast(float, e); }
                    }
                } else {
                    x[i][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0));
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int j = 0; j < P::N; ++j) acc[j] += x[i][j];
        }
    };
    const bool is_long = end - c > LONG && end >= 0;
    if (lane == 0) {
        run_end[w] = is_long ? end : -1;
        run_id[w] = id;
    }
    if (end >= 0 && !is_long) {
        const int col = (seg * 64 + lane) * P::N;
        P r;
        total(c, c + 1, end, true, col, r.x);
        if (col < C) {
#pragma unroll
            for (int j = 0; j < P::N; ++j) r.x[j] *= scale;
            r.store(dw, (int64_t)id * C + col);
        }
    }
    __syncthreads();
    for (int i = 0; i < JOIN; ++i) {
        const int64_t last = run_end[i];
        if (last < 0) continue;                                            // the same for all waves
        const int64_t uu = u0 + i, cc = uu / nseg, each = (last - cc + JOIN - 1) / JOIN, k0 = cc + 1 + w * each, k1 = k0 + each - 1 < last ? k0 + each - 1 : last;
        const int col = ((int)(uu - cc * nseg) * 64 + lane) * P::N;
        P r;
        total(cc, k0, k1, w == 0, col, r.x);
#pragma unroll
        for (int j = 0; j < P::N; ++j) sums[w][64 * j + lane] = r.x[j];
        __syncthreads();
        if (w == 0 && col < C) {
#pragma unroll
            for (int j = 0; j < P::N; ++j) {
                for (int k = 1; k < JOIN; ++k) r.x[j] += sums[k][64 * j + lane];
                r.x[j] *= scale;
            }
            r.store(dw, (int64_t)run_id[i] * C + col);
        }
        __syncthreads();
    }
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
    // positions of a wave: short ones while there are few (340 tokens: 8 instead of 32 take 8 -> 4 us), about 4096 chunks of many tokens
    const int64_t few = T / 2048 / 8 * 8, many = T / 4096 / 8 * 8;
    p.chunk = (int)(many > 32 ? many : few > 32 ? 32 : few < 8 ? 8 : few);
    p.chunks = (T + p.chunk - 1) / p.chunk;
    p.pairs = up16((size_t)T * 8);
    p.counts = 2 * p.pairs;
    p.parts = p.counts + up16(((size_t)DIGITS * up4(p.nblk) + 4) * 4);
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
    const int64_t least = (T >> 23) + 1;                                   // more rows a block where there are more than 2^23 of them
    const int rows = (int)(cpr >= 1024 || 1024 / cpr < least ? least : 1024 / cpr);
    const int64_t blocks = (T + rows - 1) / rows;
    if (blocks >= 1 << 24) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);         // 2^32 threads a launch
    if (i64) FAVAE_KLAUNCH((embed_fwd_kernel<TY, VEC, int64_t>), dim3((unsigned)blocks), dim3(256), 0, s, ids, w, ws, V, out, T, C, cpr, rows, scale);
    else FAVAE_KLAUNCH((embed_fwd_kernel<TY, VEC, int32_t>), dim3((unsigned)blocks), dim3(256), 0, s, ids, w, ws, V, out, T, C, cpr, rows, scale);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}

template <int TY, bool VEC>
int go_sums(const uint2* sorted, const unsigned* valid, const void* dout, void* dw, float* part, int64_t T, int C, const Plan& p, float scale, hipStream_t s) {
    const int per = 64 * Piece<TY, VEC>::N, nseg = (C + per - 1) / per;
    const int64_t blocks = (p.chunks * nseg + 3) / 4;
    FAVAE_KLAUNCH((embed_sum_kernel<TY, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, sorted, valid, dout, dw, part, T, C, p.chunk, nseg, scale);
    FAVAE_CHECK_LAUNCH();
    if (p.chunks > 1) {
        FAVAE_KLAUNCH((embed_join_kernel<TY, VEC>), dim3((unsigned)((p.chunks * nseg + JOIN - 1) / JOIN)), dim3(64 * JOIN), 0, s, sorted, valid, dw, (const float*)part, T, C, p.chunk,
                      p.chunks, nseg, scale);
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
    const bool vec = vec_ok(dtype, C, 0, dout, dweight);
    const int per = vec ? (dtype == F32 ? 256 : 512) : 64;                 // columns of a wave in the sums
    if ((p.chunks * ((C + per - 1) / per) + 3) / 4 >= 1 << 24) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);      // 2^32 threads a launch
    if (ws_bytes < p.total) return favae_prof_fail_(FAVAE_ERR_WORKSPACE);
    const hipStream_t s = (hipStream_t)stream;
    uint2* const buf[2] = {(uint2*)ws, (uint2*)((char*)ws + p.pairs)};
    unsigned* const count = (unsigned*)((char*)ws + p.counts);
    unsigned* const valid = count + (size_t)DIGITS * up4(p.nblk);
    float* const part = (float*)((char*)ws + p.parts);
    const int64_t dw_bytes = V * C * (dtype == F32 ? 4 : 2);
    const int64_t zb = (dw_bytes + 65535) / 65536;                         // workgroups that clear the gradient
    const int zeros = (int)(zb > 2048 ? 2048 : zb);
    const uint2* sorted = buf[0];
    if (T <= SMALL) {
        if (ids_are_64bit) FAVAE_KLAUNCH((embed_sort_small_kernel<int64_t>), dim3(1 + zeros), dim3(256), 0, s, ids, buf[0], (int)T, V, padding_idx, p.passes, valid, dweight, dw_bytes);
        else FAVAE_KLAUNCH((embed_sort_small_kernel<int32_t>), dim3(1 + zeros), dim3(256), 0, s, ids, buf[0], (int)T, V, padding_idx, p.passes, valid, dweight, dw_bytes);
        FAVAE_CHECK_LAUNCH();
    } else {
        const dim3 g0(zeros > p.nblk ? zeros : p.nblk), g(p.nblk), t(256);
        for (int k = 0; k < p.passes; ++k) {
            const uint2* in = buf[(k + 1) & 1];
            uint2* out = buf[k & 1];
            if (k) {
                FAVAE_KLAUNCH((embed_count_kernel<int32_t, false>), g, t, 0, s, ids, in, T, V, padding_idx, p.tpb, p.nblk, k, count, valid, dweight, dw_bytes);
                FAVAE_CHECK_LAUNCH();
                FAVAE_KLAUNCH((embed_scatter_kernel<int32_t, false>), g, t, 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, count, valid);
            } else if (ids_are_64bit) {
                FAVAE_KLAUNCH((embed_count_kernel<int64_t, true>), g0, t, 0, s, ids, in, T, V, padding_idx, p.tpb, p.nblk, k, count, valid, dweight, dw_bytes);
                FAVAE_CHECK_LAUNCH();
                FAVAE_KLAUNCH((embed_scatter_kernel<int64_t, true>), g, t, 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, count, valid);
            } else {
                FAVAE_KLAUNCH((embed_count_kernel<int32_t, true>), g0, t, 0, s, ids, in, T, V, padding_idx, p.tpb, p.nblk, k, count, valid, dweight, dw_bytes);
                FAVAE_CHECK_LAUNCH();
                FAVAE_KLAUNCH((embed_scatter_kernel<int32_t, true>), g, t, 0, s, ids, in, out, T, V, padding_idx, p.tpb, p.nblk, k, count, valid);
            }
            FAVAE_CHECK_LAUNCH();
            sorted = out;
        }
    }
#define GO(TY)                                                                                      \
    return vec ? go_sums<TY, true>(sorted, valid, dout, dweight, part, T, C, p, scale, s)              \
               : go_sums<TY, false>(sorted, valid, dout, dweight, part, T, C, p, scale, s)
    if (dtype == F32) GO(F32);
    if (dtype == BF16) GO(BF16);
    GO(F16);
#undef GO
}
