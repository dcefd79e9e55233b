// A word of page-locked host memory for each device, which kernels write when a bounded wait gives up and which the host reads. Made by the first call that asks for it;
// there is one, whichever threads ask at a time, and it may be asked for beside a stream that is being captured, in any mode.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <mutex>

template <int DEVICES>
class StatusWords {
public:
    cudaError_t get(int device, int** word) {
        int* w = words_[device].load(std::memory_order_acquire);
        if (!w) {
            std::lock_guard<std::mutex> lock(mutex_);
            w = words_[device].load(std::memory_order_relaxed);
            if (!w) {
                void* p = nullptr;
                cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
                cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
                if (e != cudaSuccess) return e;
                const cudaError_t made = cudaHostAlloc(&p, sizeof(int), cudaHostAllocDefault);
                e = cudaThreadExchangeStreamCaptureMode(&mode);
                if (made != cudaSuccess || e != cudaSuccess) return made != cudaSuccess ? made : e;
                w = static_cast<int*>(p);
                *w = 0;
                words_[device].store(w, std::memory_order_release);
            }
        }
        *word = w;
        return cudaSuccess;
    }

private:
    std::mutex mutex_;
    std::atomic<int*> words_[DEVICES] = {};
};
