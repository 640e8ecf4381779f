// Attention of chunks over the 8-bit cache, fp16 queries (kv8_chunk.h).
#include "kv8_chunk.h"

template int pkv::launch_kv8_chunk<_Float16>(const pkv::Kv8Params& p, hipStream_t stream);
