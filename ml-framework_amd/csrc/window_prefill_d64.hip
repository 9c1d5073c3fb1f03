// window_prefill_d64.hip -- head_dim 64 instantiations of the chunks' attention over a window and sinks.
#define PA_WINDOW_INSTANTIATE
#include <type_traits>

#include "window_prefill.h"

template void pa::launch_window_prefill<64>(const pa::WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
