// The kernels of norms.hpp for one pair of types (MINT_NORM_PAIR), in a translation unit of their own, so that the pairs compile side by side.
#include "norms.hpp"

namespace mint {

#define MINT_DEFINE(name, S, T)                                                                      \
    int launch_join_##name(const JoinArgs& a, hipStream_t s) { return go_join<S, T>(a, s); }         \
    int launch_join_grad_##name(const JoinGradArgs& a, bool bias, hipStream_t s) { return go_join_grad<S, T>(a, bias, s); }
#if MINT_NORM_PAIR == 0
MINT_DEFINE(f16, DT_F16, DT_F16)
#elif MINT_NORM_PAIR == 1
MINT_DEFINE(bf16, DT_BF16, DT_BF16)
#elif MINT_NORM_PAIR == 2
MINT_DEFINE(f32, DT_F32, DT_F32)
#elif MINT_NORM_PAIR == 3
MINT_DEFINE(f32_f16, DT_F32, DT_F16)
#else
MINT_DEFINE(f32_bf16, DT_F32, DT_BF16)
#endif

}  // namespace mint
