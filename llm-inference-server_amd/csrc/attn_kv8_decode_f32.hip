// Decode attention over the 8-bit cache, fp32 queries (kv8_decode.h).
#include "kv8_decode.h"

template int pkv::launch_kv8_decode<float>(const pkv::Kv8Params& p, hipStream_t stream);
