// libreax_decode.so -- what a serving step reads and writes (no counterpart in the reference): the quantised key/value
// cache, attention over its pages (the sequences' own and a prefix that a batch shares), and the gated delta rule with a
// carried state, sm_100a.  ABI: the EXTENSIONS of include/reax_abi.h.
#include "delta_chunk.cuh"
#include "kvcache.cuh"
#include "paged_launch.cuh"

REAX_DEFINE_STATUS_EXPORT()
REAX_DEFINE_KV_EXPORTS()
REAX_DEFINE_DELTA_STATE_EXPORT()
