// Host-side services that the translation units of the library share; defined in rs_sampler.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace rs {

struct HostDevice {
    int sms;           // multiprocessors of the current device
    int smem_optin;    // most dynamic shared memory of a block
    int* mirror;       // host word that kernels copy a non-zero status to (rs_set_status_mirror), or null
};

int host_device(HostDevice* out);                       // of the current device; RS_OK or RS_ERR_CUDA
int host_cuda_fail(cudaError_t e, const char* what);    // keeps the message for rs_last_cuda_error, returns RS_ERR_CUDA
void host_count_launch();                               // counts one kernel for rs_kernel_launch_count
uint32_t host_wait_polls();                             // poll limit of the kernels' bounded waits
int host_status_word(int** out);                        // device address of the word that rs_logprobs_status reads (rs_logprobs.cu)

}  // namespace rs
