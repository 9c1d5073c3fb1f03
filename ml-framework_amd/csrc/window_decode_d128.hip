// window_decode_d128.hip -- head_dim 128 instantiations of the attention over a window and sinks.
#define PA_WINDOW_INSTANTIATE
#include "window_decode.h"

template void pa::launch_window_decode<128>(const pa::WindowArgs&, int, bool, hipStream_t);
