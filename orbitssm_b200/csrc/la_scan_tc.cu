#include "common.cuh"
#include "la_args.h"
namespace orbit {
bool la_tc_serves(const LaArgs&, bool, int) { return false; }
int la_tc_launch(const LaArgs&, bool, cudaStream_t) { return OK; }
int la_tc_segments(const LaArgs&, bool, int*) { return 1; }
}
