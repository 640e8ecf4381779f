// Attention of chunks over the 8-bit cache, bf16 queries (kv8_chunk.h).
#include "kv8_chunk.h"

template int pkv::launch_kv8_chunk<pkv::bf16_t>(const pkv::Kv8Params& p, hipStream_t stream);
