// The gated delta rule's chunked kernels for float storage.
#include "seq_delta.h"

namespace snnseq {
SNNSEQ_DEFINE_DELTA(f32, float)
}  // namespace snnseq
