// Decode attention over the 8-bit cache, fp16 queries (kv8_decode.h).
#include "kv8_decode.h"

template int pkv::launch_kv8_decode<_Float16>(const pkv::Kv8Params& p, hipStream_t stream);
