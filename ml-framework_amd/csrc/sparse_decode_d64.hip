// sparse_decode_d64.hip -- head_dim 64 instantiations of the attention over selected blocks.
#define PA_SPARSE_INSTANTIATE
#include "sparse_decode.h"

template void pa::launch_sparse_decode<64>(const pa::SparseArgs&, int, bool, hipStream_t);
