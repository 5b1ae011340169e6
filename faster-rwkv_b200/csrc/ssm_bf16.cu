#define FRB_SSM_KERNELS
#include "ssm.cuh"

template cudaError_t frb::launch_ssm_seq<__nv_bfloat16>(const SsmArgs &, const SeqTable &, cudaStream_t);
