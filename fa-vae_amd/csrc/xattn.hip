// Cross attention, host side: argument checks, the choice of a kernel's tiling and of the splits, the three passes of the backward.
#include "xattn.h"

namespace {
using namespace xattn;

int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

struct Plan {
    int few, tiles, nsplit, span;          // few: 0 many rows, 1 up to 64, 2 up to 16, 3 many rows over few keys (forward)
};

// Splits the streamed axis of n elements into spans (multiples of 64, none under 128): the number of splits with the smallest estimate.
// `base` workgroups exist without splits, `fit` of them run together on a CU, `tau` us is what one alone takes for 64 elements (and about
// as much to start); two together take 1.5 times as long, three 1.7 times; a join takes 4 us, reads `bytes` a split at 7 TB/s and waits
// `wait` us a split: 0.042 in the sums of the backward pass (dq of 512 values: 31 us for 683 splits, 9 for 157; dk and dv make two),
// 0.02 in the forward one (14 us for 512 splits of 8 rows).
// Measured (us): fp32, 192 workgroups of 1500 keys x 64 columns: 104 in one span, 79 + 6 in 2, 83 + 6 in 3, 71 + 7 in 4, 75 + 10 in 8;
// fp32, 40 of 5036 x 128: 801, 410 + 5, 283 + 5, 227 + 5, 124 + 5 in 8, 102 + 10 in 12; fp16, 288 of 515 x 80: 29, 28 + 8 in 2.
void split_axis(int64_t base, int64_t n, int fit, double tau, double bytes, double wait, Plan& p) {
    static const double together[4] = {0.0, 1.0, 1.5, 1.7};
    const int64_t most = n / 128 < 1 ? 1 : n / 128 < MOST_SPLITS ? n / 128 : MOST_SPLITS, slots = 256 * (int64_t)fit;
    double best = 0.0;
    for (int64_t s = 1; s <= most && (s == 1 || base * s <= 4 * slots); s += 1 + s / 16) {
        const int64_t span = up((n + s - 1) / s, 64), ns = (n + span - 1) / span, full = base * ns / slots, rest = base * ns % slots;
        const double t = (span / 64 + 1) * tau * (full * together[fit] + together[(rest + 255) / 256]) + (ns > 1 ? 4.0 + ns * (bytes / 7e6 + wait) : 0.0);
        if (s > 1 && t >= best) continue;
        best = t;
        p.span = (int)span;
        p.nsplit = (int)ns;
    }
}
// about `want` workgroups instead: few rows over many keys, bound by the keys' bytes
void split_even(int64_t base, int64_t n, int step, int least, int64_t want, Plan& p) {
    const int64_t most = n / least < 1 ? 1 : n / least < MOST_SPLITS ? n / least : MOST_SPLITS, w = (want + base - 1) / base;
    const int64_t s = w < most ? w : most, span = up((n + s - 1) / s, step);
    p.span = (int)span;
    p.nsplit = (int)((n + span - 1) / span);
}

int dim_pad(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

Plan plan_fwd(const favae_xattn_desc* d) {
    const int64_t R = (int64_t)d->H / d->Hkv * d->Lq, heads = (int64_t)d->B * d->Hkv;
    const bool f32 = d->dtype == F32;
    Plan p{};
    if (R <= 64) {
        p.few = R <= 16 ? 2 : 1;
        p.tiles = (int)((R + 31) / 32);
        split_even(p.tiles * heads, d->Lk, f32 && dim_pad(d->D) > 64 ? 64 : 128, 256, 512, p);   // measured on 32 heads x 30011 keys: 256, 1024 are slower
    } else if (d->Lk <= (f32 ? 96 : 128) && (!f32 || d->D <= 64)) {
        p.few = 3;
        const int64_t tiles = (R + 127) / 128, want = (512 + heads - 1) / heads, wgs = want < tiles ? want : tiles;   // two workgroups a CU
        const int64_t span = (tiles + wgs - 1) / wgs;                      // row tiles of a workgroup
        p.nsplit = 1;
        p.span = (int)(span * 128);
        p.tiles = (int)((tiles + span - 1) / span);
    } else {
        p.tiles = (int)((R + 127) / 128);
        split_axis(p.tiles * heads, d->Lk, !f32 && d->D <= 64 ? 3 : 2, (f32 ? 2.2 : 0.6) * dim_pad(d->D) / 32, 4.0 * R * heads * d->D, 0.02, p);
    }
    return p;
}
Plan plan_dq(const favae_xattn_desc* d) {
    const int64_t R = (int64_t)d->H / d->Hkv * d->Lq, heads = (int64_t)d->B * d->Hkv;
    Plan p{};
    p.tiles = (int)((R + 127) / 128);
    const bool f32 = d->dtype == F32;
    split_axis(p.tiles * heads, d->Lk, f32 ? (d->D > 64 ? 1 : 2) : d->D <= 64 ? 3 : 2, (f32 ? 2.4 : 0.75) * dim_pad(d->D) / 32, 4.0 * R * heads * d->D,
               0.042, p);
    return p;
}
Plan plan_dkv(const favae_xattn_desc* d) {
    const int64_t R = (int64_t)d->H / d->Hkv * d->Lq, heads = (int64_t)d->B * d->Hkv;
    Plan p{};
    p.tiles = (d->Lk + 127) / 128;
    const bool f32 = d->dtype == F32;
    split_axis(p.tiles * heads, R, f32 && d->D > 64 ? 1 : 2, (f32 ? 3.9 : 1.1) * dim_pad(d->D) / 32, 8.0 * heads * d->Lk * d->D, 0.084, p);
    return p;
}

float args_c(const favae_xattn_desc* d) { return (float)((double)d->scale * 1.4426950408889634); }      // scale in powers of two

// sizes and strides the kernels can take; the byte range of an element type's strides is the caller's memory
bool ok_desc(const favae_xattn_desc* d) {
    if (!d || d->B < 1 || d->Lq < 1 || d->Lk < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv || d->D < 8 || d->D > 128 || d->D % 8) return false;
    if (d->dtype < F32 || d->dtype > F16 || !(d->scale > 0.f) || !(args_c(d) < INFINITY)) return false;
    const int64_t R = (int64_t)d->H / d->Hkv * d->Lq, heads = (int64_t)d->B * d->Hkv;
    if (R > (1 << 30) || d->Lk > (1 << 30) || heads > (1 << 24)) return false;
    if (((R + 31) / 32 > (d->Lk + 127) / 128 ? (R + 31) / 32 : (d->Lk + 127) / 128) * heads >= (1 << 24)) return false;   // 2^32 threads a launch
    const int64_t unit = d->dtype == F32 ? 4 : 8;                          // 16-byte accesses
    for (int64_t s : {d->q_sb, d->q_sl, d->q_sh, d->k_sb, d->k_sl, d->k_sh, d->v_sb, d->v_sl, d->v_sh})
        if (s < 0 || s % unit) return false;
    // rows follow one another and 128 of them span less than 2^31 bytes (those of the dense outputs and of dout too)
    if ((int64_t)d->H * d->D * (16 / unit) >= (1 << 24)) return false;
    for (int64_t s : {d->q_sl, d->k_sl, d->v_sl})
        if (s < d->D || s * (16 / unit) >= (1 << 24)) return false;
    return true;
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

Args args_of(const favae_xattn_desc* d, const void* q, const void* k, const void* v, const uint8_t* pad) {
    Args a{};
    a.q = q; a.k = k; a.v = v; a.pad = pad;
    a.q_b = d->q_sb; a.q_l = d->q_sl; a.q_h = d->q_sh;
    a.k_b = d->k_sb; a.k_l = d->k_sl; a.k_h = d->k_sh;
    a.v_b = d->v_sb; a.v_l = d->v_sl; a.v_h = d->v_sh;
    a.pad_b = d->pad_sb;
    a.B = d->B; a.Lq = d->Lq; a.Lk = d->Lk; a.H = d->H; a.Hkv = d->Hkv; a.G = d->H / d->Hkv; a.D = d->D;
    a.R = a.G * a.Lq;
    a.scale = d->scale;
    a.c = args_c(d);
    return a;
}
void use(Args& a, const Plan& p) { a.tiles = p.tiles; a.nsplit = p.nsplit; a.span = p.span; }

int64_t rows_of(const favae_xattn_desc* d) { return (int64_t)d->B * d->H * d->Lq; }

int run_fwd(int ty, const Args& a, const Plan& p, hipStream_t s) {
    return ty == F32 ? launch_fwd<F32>(a, p.few, s) : ty == BF16 ? launch_fwd<BF16>(a, p.few, s) : launch_fwd<F16>(a, p.few, s);
}
int run_join_fwd(int ty, const Args& a, hipStream_t s) {
    return ty == F32 ? launch_join_fwd<F32>(a, s) : ty == BF16 ? launch_join_fwd<BF16>(a, s) : launch_join_fwd<F16>(a, s);
}
int run_dq(int ty, const Args& a, hipStream_t s) {
    return ty == F32 ? launch_bwd_dq<F32>(a, s) : ty == BF16 ? launch_bwd_dq<BF16>(a, s) : launch_bwd_dq<F16>(a, s);
}
int run_dkv(int ty, const Args& a, hipStream_t s) {
    return ty == F32 ? launch_bwd_dkv<F32>(a, s) : ty == BF16 ? launch_bwd_dkv<BF16>(a, s) : launch_bwd_dkv<F16>(a, s);
}
int run_join_sum(int ty, const float* part, void* out, int64_t n, int ns, hipStream_t s) {
    return ty == F32 ? launch_join_sum<F32>(part, out, n, ns, s) : ty == BF16 ? launch_join_sum<BF16>(part, out, n, ns, s)
                                                                               : launch_join_sum<F16>(part, out, n, ns, s);
}

}  // namespace

extern "C" size_t favae_xattn_fwd_workspace(const favae_xattn_desc* d) {
    if (!ok_desc(d)) return 0;
    const Plan p = plan_fwd(d);
    return p.nsplit > 1 ? (size_t)(p.nsplit * rows_of(d) * (d->D + 1)) * 4 : 0;
}

extern "C" int favae_xattn_fwd(const favae_xattn_desc* d, const void* q, const void* k, const void* v, const uint8_t* key_padding_mask,
                               void* o, float* o32, float* lse, void* ws, size_t ws_bytes, favae_stream_t stream) {
    FAVAE_REQUIRE(d && q && k && v && o);
    if (!ok_desc(d) || !aligned(q) || !aligned(k) || !aligned(v) || !aligned(o) || !aligned(o32) || !aligned(ws))
        return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    const Plan p = plan_fwd(d);
    if (p.nsplit > 1 && (!ws || ws_bytes < favae_xattn_fwd_workspace(d))) return favae_prof_fail_(FAVAE_ERR_WORKSPACE);
    Args a = args_of(d, q, k, v, key_padding_mask);
    use(a, p);
    a.o = o; a.o32 = o32; a.lse = lse;
    if (p.nsplit > 1) {
        a.part = (float*)ws;
        a.part_lse = a.part + p.nsplit * rows_of(d) * d->D;
    }
    FAVAE_PROF_NOTE(4.0 * rows_of(d) * d->Lk * d->D, 0);
    if (int rc = run_fwd(d->dtype, a, p, (hipStream_t)stream)) return rc;
    return p.nsplit > 1 ? run_join_fwd(d->dtype, a, (hipStream_t)stream) : FAVAE_OK;
}

extern "C" size_t favae_xattn_bwd_workspace(const favae_xattn_desc* d) {
    if (!ok_desc(d)) return 0;
    const Plan pq = plan_dq(d), pk = plan_dkv(d);
    const int64_t nq = pq.nsplit > 1 ? pq.nsplit * rows_of(d) * d->D : 0;
    const int64_t nk = pk.nsplit > 1 ? 2 * (int64_t)pk.nsplit * d->B * d->Lk * d->Hkv * d->D : 0;
    return (size_t)(up(rows_of(d), 4) + (nq > nk ? nq : nk)) * 4;
}

extern "C" int favae_xattn_bwd(const favae_xattn_desc* d, const void* q, const void* k, const void* v, const uint8_t* key_padding_mask,
                               const float* o32, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* ws,
                               size_t ws_bytes, favae_stream_t stream) {
    FAVAE_REQUIRE(d && q && k && v && o32 && lse && dout && dq && ws && !dk == !dv);
    for (const void* p : {q, k, v, (const void*)o32, dout, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)ws})
        if (!aligned(p)) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    if (!ok_desc(d)) return favae_prof_fail_(FAVAE_ERR_UNSUPPORTED);
    if (ws_bytes < favae_xattn_bwd_workspace(d)) return favae_prof_fail_(FAVAE_ERR_WORKSPACE);
    const hipStream_t s = (hipStream_t)stream;
    Args a = args_of(d, q, k, v, key_padding_mask);
    a.dout = dout;
    a.d_h = d->D; a.d_l = (int64_t)d->H * d->D; a.d_b = a.d_l * d->Lq;
    a.o32 = const_cast<float*>(o32);
    a.lse = const_cast<float*>(lse);
    a.delta = (float*)ws;
    a.part = a.delta + up(rows_of(d), 4);
    a.dq = dq; a.dk = dk; a.dv = dv;
    const Plan pq = plan_dq(d);
    use(a, pq);
    FAVAE_PROF_NOTE(6.0 * rows_of(d) * d->Lk * d->D, 0);
    if (int rc = run_dq(d->dtype, a, s)) return rc;
    if (pq.nsplit > 1)
        if (int rc = run_join_sum(d->dtype, a.part, dq, rows_of(d) * d->D, pq.nsplit, s)) return rc;
    if (!dk) return FAVAE_OK;
    const Plan pk = plan_dkv(d);
    const int64_t n = (int64_t)d->B * d->Lk * d->Hkv * d->D;
    use(a, pk);
    a.part2 = a.part + pk.nsplit * n;
    FAVAE_PROF_NOTE(8.0 * rows_of(d) * d->Lk * d->D, 0);
    if (int rc = run_dkv(d->dtype, a, s)) return rc;
    if (pk.nsplit > 1) {
        if (int rc = run_join_sum(d->dtype, a.part, dk, n, pk.nsplit, s)) return rc;
        return run_join_sum(d->dtype, a.part2, dv, n, pk.nsplit, s);
    }
    return FAVAE_OK;
}
