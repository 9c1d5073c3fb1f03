// window_prefill_d32.hip -- head_dim 32 instantiations of the chunks' attention over a window and sinks.
#define PA_WINDOW_INSTANTIATE
#include <type_traits>

#include "window_prefill.h"

template void pa::launch_window_prefill<32>(const pa::WindowPrefillArgs&, int, bool, bool, uint32_t, hipStream_t);
