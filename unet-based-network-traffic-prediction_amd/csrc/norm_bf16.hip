#include "norm_impl.h"
namespace mi {
int launch_gn_fwd_bf16(const NormArgs& a, const Slab* sl, hipStream_t s) { return launch_gn_fwd_t<__bf16>(a, sl, s); }
int launch_gn_bwd_bf16(const NormArgs& a, const Slab* sl, hipStream_t s) { return launch_gn_bwd_t<__bf16>(a, sl, s); }
}
