#include "tq_paged_few.h"

int tq_paged_few_launch_d256(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors) { return launch_paged_few<256>(ipbk, ipbv, grid, s, a, vectors); }
