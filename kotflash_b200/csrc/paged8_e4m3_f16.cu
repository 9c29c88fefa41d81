// K9's kernels for e4m3 pages with fp16 queries.
#include "paged8_decode.cuh"

int kf::paged8_launch_e4m3_f16(const kf::Paged8Launch& l) { return dispatch<false, false>(l); }
