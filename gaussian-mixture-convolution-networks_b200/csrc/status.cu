// Status strings, the per-thread CUDA error message and the device check word reader.
#include <mutex>

#include "common.cuh"

namespace gmc {
namespace {
thread_local cudaError_t t_last_error = cudaSuccess;
}
void set_last_cuda_error(cudaError_t e) { t_last_error = e; }
}  // namespace gmc

// one check word per translation unit that owns kernels
int gmc_tu_check_eval_inversed(int** word);
int gmc_tu_check_small_ops(int** word);
int gmc_tu_check_lbvh(int** word);
int gmc_tu_check_mhem_fit(int** word);
int gmc_tu_check_convolution(int** word);
int gmc_tu_check_convolution_fitting(int** word);
int gmc_tu_check_relu_fixed_point(int** word);
int gmc_tu_check_log_probabilities(int** word);
int gmc_tu_check_newton_schulz(int** word);

extern "C" const char* gmc_status_string(int status) {
    switch (status) {
        case GMC_OK: return "ok";
        case GMC_ERR_BAD_DIMS: return "bad dimensions: D must be 2 or 3 and every extent positive and within its limit";
        case GMC_ERR_BAD_BROADCAST: return "xes must have a batch and layer extent of one or equal to the mixture's";
        case GMC_ERR_NULL_POINTER: return "a required pointer is NULL";
        case GMC_ERR_UNSUPPORTED: return "unsupported parameter value";
        case GMC_ERR_CUDA: return "CUDA runtime error";
        case GMC_ERR_DEVICE_CHECK: return "a device-side check failed";
        case GMC_ERR_BUILTIN_SCRATCH:
            return "problem exceeds the built-in scratch of the no-allocation entry point (n_mixtures * n_components > "
                   "2^20); use the entry point that takes caller scratch";
        case GMC_ERR_WORKSPACE: return "the workspace is smaller than the entry point's ..._workspace_bytes asks for";
        default: return "unknown status";
    }
}

extern "C" const char* gmc_last_cuda_error(void) {
    return gmc::t_last_error == cudaSuccess ? "" : cudaGetErrorString(gmc::t_last_error);
}

extern "C" const char* gmc_version(void) { return "0.1"; }

static int read_all_check_words(int* word_out);

extern "C" int gmc_sync_and_check(void* stream) {
    GMC_CUDA_TRY(cudaStreamSynchronize(gmc::as_stream(stream)));
    int word = 0;
    if (int s = read_all_check_words(&word)) return s;
    return word != 0 ? GMC_ERR_DEVICE_CHECK : GMC_OK;
}

extern "C" int gmc_device_check_word(int* word_out) {
    if (!word_out) return GMC_ERR_NULL_POINTER;
    *word_out = 0;
    GMC_CUDA_TRY(cudaDeviceSynchronize());
    return read_all_check_words(word_out);
}

namespace gmc {
namespace {
constexpr int (*kUnits[])(int**) = {gmc_tu_check_eval_inversed,
                                    gmc_tu_check_small_ops,
                                    gmc_tu_check_lbvh,
                                    gmc_tu_check_mhem_fit,
                                    gmc_tu_check_convolution,
                                    gmc_tu_check_convolution_fitting,
                                    gmc_tu_check_relu_fixed_point,
                                    gmc_tu_check_log_probabilities,
                                    gmc_tu_check_newton_schulz};
constexpr int kWords = int(sizeof(kUnits) / sizeof(kUnits[0]));
static_assert(kWords <= 32, "one lane per word");
struct CheckWords {
    int* word[kWords];
};
__device__ int g_all_words;

// One warp reads and clears all words: with nothing to wait for gmc_sync_and_check takes 26 us, where a copy for each of nine words
// took 119.
__global__ void collect_check_words(CheckWords w) {
    const int lane = threadIdx.x;
    const int all = __reduce_or_sync(0xffffffffu, unsigned(lane < kWords ? atomicExch(w.word[lane], 0) : 0));
    if (lane == 0) g_all_words = all;
}
}  // namespace
}  // namespace gmc

static int read_all_check_words(int* word_out) {
    gmc::CheckWords words;
    for (int i = 0; i < gmc::kWords; ++i)
        if (int s = gmc::kUnits[i](&words.word[i])) return s;
    static std::mutex one_at_a_time;                                  // g_all_words is one call's until it is copied
    std::lock_guard<std::mutex> lock(one_at_a_time);
    void* arguments[] = {&words};
    GMC_CUDA_TRY(cudaLaunchKernel(reinterpret_cast<const void*>(gmc::collect_check_words), dim3(1), dim3(32), arguments, 0, nullptr));
    int all = 0;
    GMC_CUDA_TRY(cudaMemcpyFromSymbol(&all, gmc::g_all_words, sizeof(int)));
    *word_out |= all;
    return GMC_OK;
}
