// sparse_decode_d128.hip -- head_dim 128 instantiations of the attention over selected blocks.
#define PA_SPARSE_INSTANTIATE
#include "sparse_decode.h"

template void pa::launch_sparse_decode<128>(const pa::SparseArgs&, int, bool, hipStream_t);
