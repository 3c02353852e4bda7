// The gated delta rule's chunked kernels for bf16_t storage.
#include "seq_delta.h"

namespace snnseq {
SNNSEQ_DEFINE_DELTA(bf16, bf16_t)
}  // namespace snnseq
