// The entry points of include/snnlib_seq.h that belong to no operator.
#include "snnlib_seq.h"

extern "C" int snnseq_abi_version(void) { return SNNSEQ_ABI_VERSION; }
