// Launches of the cross attention kernels of one element type.
#pragma once
#include "xattn.h"

namespace xattn {

// more than 64 KB of dynamic LDS has to be asked for
template <typename F>
inline int ready(F kern, size_t lds) {
    return lds <= 65536 || hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) == hipSuccess
               ? FAVAE_OK : favae_prof_fail_(FAVAE_ERR_LAUNCH);
}

template <int TY, int DP, bool KEYW>
int go_fwd(const Args& a, hipStream_t s) {
    using C = FwdCfg<TY, DP, KEYW>;
    if (int rc = ready(fwd_kernel<TY, DP, KEYW>, C::LDS)) return rc;
    FAVAE_KLAUNCH((fwd_kernel<TY, DP, KEYW>), dim3((unsigned)(a.tiles * a.nsplit) * a.B * a.Hkv), dim3(C::NT), C::LDS, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}
template <int TY, int DP>
int go_token(const Args& a, hipStream_t s) {
    using C = TokCfg<TY, DP>;
    if (int rc = ready(fwd_token_kernel<TY, DP>, C::LDS)) return rc;
    FAVAE_KLAUNCH((fwd_token_kernel<TY, DP>), dim3((unsigned)a.nsplit * a.B * a.Hkv), dim3(C::NT), C::LDS, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}
template <int TY, int DP>
int go_short(const Args& a, hipStream_t s) {
    using C = ShortCfg<TY, DP>;
    if (int rc = ready(fwd_short_kernel<TY, DP>, C::LDS)) return rc;
    FAVAE_KLAUNCH((fwd_short_kernel<TY, DP>), dim3((unsigned)a.tiles * a.B * a.Hkv), dim3(C::NT), C::LDS, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}
template <int TY, int DP>
int go_fwd_dp(const Args& a, int few, hipStream_t s) {
    if constexpr (ShortCfg<TY, DP>::OK) {
        if (few == 3) return go_short<TY, DP>(a, s);
    }
    return few == 2 ? go_token<TY, DP>(a, s) : few ? go_fwd<TY, DP, true>(a, s) : go_fwd<TY, DP, false>(a, s);
}
template <int TY, int DP>
int go_dq(const Args& a, hipStream_t s) {
    using C = DqCfg<TY, DP>;
    if (int rc = ready(bwd_dq_kernel<TY, DP>, C::LDS)) return rc;
    FAVAE_KLAUNCH((bwd_dq_kernel<TY, DP>), dim3((unsigned)(a.tiles * a.nsplit) * a.B * a.Hkv), dim3(C::NT), C::LDS, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}
template <int TY, int DP>
int go_dkv(const Args& a, hipStream_t s) {
    using C = DkvCfg<TY, DP>;
    if (int rc = ready(bwd_dkv_kernel<TY, DP>, C::LDS)) return rc;
    FAVAE_KLAUNCH((bwd_dkv_kernel<TY, DP>), dim3((unsigned)(a.tiles * a.nsplit) * a.B * a.Hkv), dim3(C::NT), C::LDS, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}

template <int TY> int launch_fwd(const Args& a, int few, hipStream_t s) {
    return a.D <= 32 ? go_fwd_dp<TY, 32>(a, few, s) : a.D <= 64 ? go_fwd_dp<TY, 64>(a, few, s)
         : a.D <= 96 ? go_fwd_dp<TY, 96>(a, few, s) : go_fwd_dp<TY, 128>(a, few, s);
}
template <int TY> int launch_bwd_dq(const Args& a, hipStream_t s) {
    return a.D <= 32 ? go_dq<TY, 32>(a, s) : a.D <= 64 ? go_dq<TY, 64>(a, s) : a.D <= 96 ? go_dq<TY, 96>(a, s) : go_dq<TY, 128>(a, s);
}
template <int TY> int launch_bwd_dkv(const Args& a, hipStream_t s) {
    return a.D <= 32 ? go_dkv<TY, 32>(a, s) : a.D <= 64 ? go_dkv<TY, 64>(a, s) : a.D <= 96 ? go_dkv<TY, 96>(a, s) : go_dkv<TY, 128>(a, s);
}
template <int TY> int launch_join_fwd(const Args& a, hipStream_t s) {
    if (a.nsplit <= FEW_SPLITS) {
        const int64_t n = (int64_t)a.B * a.Hkv * a.R * (a.D / 4);
        FAVAE_KLAUNCH((join_few_kernel<TY>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
    } else FAVAE_KLAUNCH((join_fwd_kernel<TY>), dim3((unsigned)(a.B * a.Hkv) * a.R), dim3(256), 0, s, a);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}
template <int TY> int launch_join_sum(const float* part, void* out, int64_t n, int nsplit, hipStream_t s) {
    FAVAE_KLAUNCH((join_sum_kernel<TY>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, part, out, n, nsplit);
    FAVAE_CHECK_LAUNCH();
    return FAVAE_OK;
}

#define XATTN_INSTANTIATE(TY)                                                                  \
    namespace xattn {                                                                          \
    template int launch_fwd<TY>(const Args&, int, hipStream_t);                           \
    template int launch_bwd_dq<TY>(const Args&, hipStream_t);                                  \
    template int launch_bwd_dkv<TY>(const Args&, hipStream_t);                                 \
    template int launch_join_fwd<TY>(const Args&, hipStream_t);                                \
    template int launch_join_sum<TY>(const float*, void*, int64_t, int, hipStream_t);          \
    }

}  // namespace xattn
