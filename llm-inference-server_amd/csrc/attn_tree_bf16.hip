// Tree attention over bf16 pools (tree_mfma.h).
#include "tree_mfma.h"

template int pkv::launch_tree_mfma<pkv::bf16_t>(const TreeParams&, hipStream_t);
