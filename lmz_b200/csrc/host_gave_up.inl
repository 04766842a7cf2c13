// Whether a kernel has given up waiting (included by model_ops.cu).
#include <cstdint>

// 1 if the word at `d_word` on the current device is set once all that was launched there has ended, on whatever stream; the
// word is cleared then, so that what is launched from here on speaks for itself.
static int taken_word(void *d_word)
{
    uint32_t word = 0;
    CK("cudaDeviceSynchronize", cudaDeviceSynchronize());
    CK("cudaMemcpy", cudaMemcpy(&word, d_word, sizeof word, cudaMemcpyDeviceToHost));
    if (!word) return 0;
    const uint32_t none = 0;
    CK("cudaMemcpy", cudaMemcpy(d_word, &none, sizeof none, cudaMemcpyHostToDevice));
    CK("cudaDeviceSynchronize", cudaDeviceSynchronize());        // (it has arrived before anything is launched)
    return 1;
}
