// Tree attention over fp16 pools (tree_mfma.h).
#include "tree_mfma.h"

template int pkv::launch_tree_mfma<_Float16>(const TreeParams&, hipStream_t);
