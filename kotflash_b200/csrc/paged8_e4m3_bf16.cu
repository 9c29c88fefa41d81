// K9's kernels for e4m3 pages with bf16 queries.
#include "paged8_decode.cuh"

int kf::paged8_launch_e4m3_bf16(const kf::Paged8Launch& l) { return dispatch<false, true>(l); }
