#include "tq_paged_kernel.h"

int tq_paged_launch_d256(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt) { return launch_paged<256>(ipbk, ipbv, grid, s, a, qt, kt, vt); }
