// bf16 instantiations of the shared-prefix attention kernels.
#include "prefix_attn.cuh"

namespace ffai {

hipError_t launch_prefix_bf16(const PrefixParams& p, int head_dim, int parts, hipStream_t s) {
  return launch_prefix_type<kBF16>(p, head_dim, parts, s);
}

hipError_t launch_whole_bf16(const PrefixParams& p, int groups, int head_dim, int parts, hipStream_t s) {
  return launch_whole_type<kBF16>(p, groups, head_dim, parts, s);
}

}  // namespace ffai
