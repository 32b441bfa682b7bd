// Parts of the attention kernels' joins by themselves: the bounded wait, which
// takes a short limit here and reports like the kernels do, and a launch's number.
#include "qmv_attention.cuh"

namespace {

__global__ void wait_kernel(const unsigned long long *flag, unsigned long long launch, unsigned long long limit_ns, unsigned int *status)
{
    if (!qmv::flag_wait(flag, launch, limit_ns)) qmv::report(status, qmv::kStatusAttentionWait);
}

__global__ void set_kernel(unsigned long long *flag, unsigned long long launch) { qmv::flag_set(flag, launch); }

__global__ void number_kernel(unsigned long long *out, qmv::LaunchTag tag)
{
    if (threadIdx.x == 0) out[blockIdx.x] = qmv::number_of(tag);
}

}  // namespace

extern "C" int check_wait(const unsigned long long *flag, unsigned long long launch, unsigned long long limit_ns, unsigned int *status)
{
    wait_kernel<<<1, 1>>>(flag, launch, limit_ns, status);
    return (int)cudaDeviceSynchronize();
}

extern "C" int check_set(unsigned long long *flag, unsigned long long launch)
{
    set_kernel<<<1, 1>>>(flag, launch);
    return (int)cudaDeviceSynchronize();
}

extern "C" int check_number(unsigned long long *out, unsigned long long number, unsigned long long *count, int ctas, void *stream)
{
    number_kernel<<<ctas, 32, 0, (cudaStream_t)stream>>>(out, qmv::LaunchTag{number, count});
    return (int)cudaGetLastError();
}
