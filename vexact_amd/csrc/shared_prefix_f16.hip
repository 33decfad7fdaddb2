// Decode attention over shared prefixes (shared_prefix.h) for fp16 on padded head sizes. A translation
// unit of its own for compile time.
#include "shared_prefix.h"

namespace vx {

int launch_shared_prefix_f16(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, hipStream_t stream) {
  if (DKb == 64 && DVb == 64) return launch_shared_prefix<ElemF16, 64, 64, true>(p, sp, stream);
  if (DKb == 128 && DVb == 128) return launch_shared_prefix<ElemF16, 128, 128, true>(p, sp, stream);
  if (DKb == 256 && DVb == 128) return launch_shared_prefix<ElemF16, 256, 128, true>(p, sp, stream);
  if (DKb == 256 && DVb == 256) return launch_shared_prefix<ElemF16, 256, 256, true>(p, sp, stream);
  return VX_ERR_UNSUPPORTED;
}

}  // namespace vx
