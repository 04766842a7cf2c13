// Checks of csrc/host_gave_up.inl over a stand-in for the CUDA runtime (cuda_runtime.h beside this file).  Exit status 0 = they held.
#include <cstdint>
#include <cstdio>

#include "cuda_runtime.h"
#include "../../include/lmz_b200.h"

// (a copy waits for the legacy stream alone, as one does beside streams that do not block it)
static int fail_copies;
static cudaError_t cudaMemcpy(void *to, const void *from, size_t n, cudaMemcpyKind)
{
    if (fake::due(fail_copies)) return cudaErrorUnknown;
    cudaStreamSynchronize(nullptr);
    memcpy(to, from, n);
    return cudaSuccess;
}
static cudaError_t cudaDeviceSynchronize()
{
    cudaStreamSynchronize(nullptr);
    for (FakeStream *s : fake::streams) cudaStreamSynchronize(s);
    return cudaSuccess;
}

#include "../../lmz_b200/csrc/host_error.inl"
#include "../../lmz_b200/csrc/host_gave_up.inl"

#define NEED(c)                                             \
    do {                                                    \
        if (!(c)) {                                         \
            fprintf(stderr, "line %d: %s\n", __LINE__, #c); \
            return 1;                                       \
        }                                                   \
    } while (0)

int main()
{
    uint32_t word = 0, one = 1;
    cudaStream_t stream;
    cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
    NEED(taken_word(&word) == 0);
    cudaMemcpyAsync(&word, &one, sizeof one, cudaMemcpyDeviceToHost, stream);      // a kernel that gives up, still to run
    NEED(taken_word(&word) == 1);
    NEED(word == 0 && taken_word(&word) == 0);                                      // (said once)
    word = 1;
    fail_copies = 2;
    NEED(taken_word(&word) == LMZ_GPU_ECUDA && word == 1);
    NEED(taken_word(&word) == 1 && taken_word(&word) == 0);
    (void)&guarded<int, int (*)()>;
    (void)&fail_msg;
    return 0;
}
