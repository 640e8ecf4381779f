// Tree attention over fp32 pools (tree_mfma.h).
#include "tree_mfma.h"

template int pkv::launch_tree_mfma<float>(const TreeParams&, hipStream_t);
