#include "dot_attention.hpp"

namespace nts {
int dot_launch_bf16(int kind, const DotArgs &p, uint32_t nd, bool near, hipStream_t stream) { return launch_kind<Bf16>(kind, p, nd, near, stream); }
}  // namespace nts
