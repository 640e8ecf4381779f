// Decode attention over the 8-bit cache, bf16 queries (kv8_decode.h).
#include "kv8_decode.h"

template int pkv::launch_kv8_decode<pkv::bf16_t>(const pkv::Kv8Params& p, hipStream_t stream);
