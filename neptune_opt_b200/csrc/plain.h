// Marks arithmetic that kernels and host compilers share.
#pragma once

#ifdef __CUDACC__
#define NB200_PLAIN __host__ __device__ __forceinline__
#else
#define NB200_PLAIN inline
#endif
