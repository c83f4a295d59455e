#include "norm_impl.h"
namespace mi {
int launch_gn_fwd_f32(const NormArgs& a, const Slab* sl, hipStream_t s) { return launch_gn_fwd_t<float>(a, sl, s); }
int launch_gn_bwd_f32(const NormArgs& a, const Slab* sl, hipStream_t s) { return launch_gn_bwd_t<float>(a, sl, s); }
}
