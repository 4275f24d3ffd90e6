#include "tq_many_fast.h"

int tq_many_launch_d128(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt) {
    if (ipbk == 4) return launch_many_fast<128, 4>(ipbv, grid, s, a, qt, kt, vt);
    if (ipbk == 2) return launch_many_fast<128, 2>(ipbv, grid, s, a, qt, kt, vt);
    return launch_many_fast<128, 1>(ipbv, grid, s, a, qt, kt, vt);
}

int tq_many_weights_launch_d128(int ipbk, dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks) {
    if (ipbk == 4) return launch_many_weights<128, 4>(grid, s, a, blocks);
    if (ipbk == 2) return launch_many_weights<128, 2>(grid, s, a, blocks);
    return launch_many_weights<128, 1>(grid, s, a, blocks);
}
