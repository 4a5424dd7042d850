#include "kernels.cuh"
#include "paged.cuh"
namespace pyr {
int prefix_tc_split(int, int, int, int) { return 0; }
int launch_prefix_tc(const AttnWork&, void*, void*, int, int, int, int, cudaStream_t) { return -4; }
}
