#define FRB_SSM_KERNELS
#include "ssm.cuh"

template cudaError_t frb::launch_ssm_seq<float>(const SsmArgs &, const SeqTable &, cudaStream_t);
