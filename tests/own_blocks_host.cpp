// own_blocks of step_plan.h for the host.
#include "../turboquant-cuda-decode_amd/csrc/step_plan.h"

extern "C" int host_own_blocks(int max_blocks, int prefix_blocks) { return tq4::xdl::own_blocks(max_blocks, prefix_blocks); }
