// Translation unit of libwgb_b200.so for the objectives, which share device code
// among themselves and come in many types: they are compiled beside the rest.
#include "wgb_common.cuh"
#include "wgb_objectives.cu"
#include "wgb_logits.cu"
