// K9's kernels for int8 pages with bf16 queries.
#include "paged8_decode.cuh"

int kf::paged8_launch_int8_bf16(const kf::Paged8Launch& l) { return dispatch<true, true>(l); }
