// Rows (tokens of activations, channels of weights) to int8 codes and a scale each (the arithmetic: dense8.cuh).
//
// A CTA has a row: its threads hold 16 values a piece in registers, agree on the largest magnitude and write 16 codes at a time. Rows longer than what
// the threads hold are read a second time, from L2.
#include <type_traits>

#include "dense8.cuh"

namespace {

constexpr int KEEP = 2;

template <typename T>
__global__ void __launch_bounds__(1024)
quantize_rows_kernel(const T* __restrict__ x, long ldx, int cols, int whole, int8_t* __restrict__ q, long ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[32];
    dep_trigger();
    dep_wait();
    const T* row = x + (size_t)blockIdx.x * ldx;
    const int pieces = (cols + 127) / 128 * 8, step = blockDim.x;
    Piece16<T> held[KEEP];
    uint32_t most = 0u;
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const int c = threadIdx.x + k * step;
        if (c < pieces) held[k] = load16(row, c, cols, whole);
    }
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if ((int)threadIdx.x + k * step < pieces) {
            float v[16];
            widen16<T>(held[k], v);
            most = max(most, most_of(v));
        }
    for (int c = threadIdx.x + KEEP * step; c < pieces; c += step) {
        float v[16];
        widen16<T>(load16(row, c, cols, whole), v);
        most = max(most, most_of(v));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, (int)(threadIdx.x & 31) < step / 32 ? red[threadIdx.x & 31] : 0u);
    const RowScale s(most);
    uint4* out = reinterpret_cast<uint4*>(q + (size_t)blockIdx.x * ldq);
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const int c = threadIdx.x + k * step;
        if (c < pieces) {
            float v[16];
            widen16<T>(held[k], v);
            out[c] = s.codes(v, most);
        }
    }
    for (int c = threadIdx.x + KEEP * step; c < pieces; c += step) {
        float v[16];
        widen16<T>(load16(row, c, cols, whole), v);
        out[c] = s.codes(v, most);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = s.scale(most);
}

template <typename T>
int launch_rows(const void* x, long ldx, int rows, int cols, int8_t* q, long ldq, float* scale, cudaStream_t st) {
    const int whole = (((uintptr_t)x | ((uintptr_t)ldx * sizeof(T))) & 15) == 0, pieces = (cols + 127) / 128 * 8;
    // few rows: as many threads as there are pieces, so that all of a row is under way at once
    const int most = rows <= 2 * cmlb_num_sms() ? 1024 : 256;
    const int threads = pieces < most ? (pieces + 31) / 32 * 32 : most;
    CMLB_CUDA(launch_chain(quantize_rows_kernel<T>, dim3(rows), dim3(threads), 0, 1, st, static_cast<const T*>(x), ldx, cols, whole, q, ldq, scale));
    return CMLB200_OK;
}

}  // namespace

extern "C" int cmlb200_quantize_rows(const void* d_x, int dtype, long ldx, int rows, int cols, int8_t* d_q, long ldq, float* d_scale, void* stream) {
    static const char* who = "cmlb200_quantize_rows";
    CMLB_REQUIRE(d_x && d_q && d_scale && rows > 0, "%s: NULL argument or %d rows", who, rows);
    CMLB_REQUIRE(cols > 0 && cols <= kMaxCols8 && ldx >= cols, "%s: %d columns (up to %d), stride %ld", who, cols, kMaxCols8, ldx);
    CMLB_REQUIRE(ldq % 128 == 0 && ldq >= cols && ((uintptr_t)d_q & 15) == 0, "%s: codes need a stride that is a multiple of 128 (%ld) and 16-byte alignment", who, ldq);
    CMLB_REQUIRE(((uintptr_t)d_scale & 3) == 0 && ((uintptr_t)d_x & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0, "%s: pointers are not aligned to their types", who);
    cudaStream_t st = as_stream(stream);
    if (dtype == CMLB200_DT_F32) return launch_rows<float>(d_x, ldx, rows, cols, d_q, ldq, d_scale, st);
    if (dtype == CMLB200_DT_BF16) return launch_rows<__nv_bfloat16>(d_x, ldx, rows, cols, d_q, ldq, d_scale, st);
    if (dtype == CMLB200_DT_F16) return launch_rows<__half>(d_x, ldx, rows, cols, d_q, ldq, d_scale, st);
    CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    return CMLB200_EINVAL;
}
