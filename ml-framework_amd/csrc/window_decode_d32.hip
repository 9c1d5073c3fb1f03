// window_decode_d32.hip -- head_dim 32 instantiations of the attention over a window and sinks.
#define PA_WINDOW_INSTANTIATE
#include "window_decode.h"

template void pa::launch_window_decode<32>(const pa::WindowArgs&, int, bool, hipStream_t);
