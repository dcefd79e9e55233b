// Rows (tokens of activations, channels of weights) to int8 codes and a scale each (the arithmetic: dense8.cuh).
//
// A group of warps has a row: its threads hold up to KEEP pieces of 16 values, agree on the largest magnitude and write the codes. Rows longer than what they hold are read a second time,
// from L2. Few rows: a CTA of as many threads as a row has pieces, so that all of it is under way at once (one row of 4,096 bf16 1.7 us). Many: CTAs of 512 threads that have several short
// rows or one long one; with a CTA a row, starting CTAs was what took the time (2,048 rows of 4,096: 10.5 us, 7.3 so), with fewer CTAs than SMs the chain of a thread's pieces (500 rows of 4,096 4.5 us, a CTA each 3.1; 333 of 777 3.1
// and 2.0; 1,000 of 4,096 with four warps each instead of two 5.8 to 4.8).
// 4,096 rows of 28,672 bf16 60 to 79 us (4.5 to 5.8 TB/s: memory), 22,016 of 4,096 44 us (6.1 TB/s). A branch for every value next to a tie, or a division, cost more than the bytes: with those the same
// rows took 122 and 116 us, since one word in seven of a warp holds half of its row's largest number.
// Two kinds of launch behind it. Codes of a product's tokens are read behind the product's wait, so it may begin at once (`ahead`). Codes of a weight are read in front of that wait, by a product
// that the caller queues next: the public entry point lets nothing begin before all CTAs have ended, what they wrote in sight of the device and of its asynchronous copies. That
// fence costs 0.5 us a call (one row of 4,096 2.2 us, 500 3.8), a tenth where memory bounds it (4,096 of 28,672 66); an end without it would promise nothing to reads in front of a wait.
// Rows that do not lie on 16-byte boundaries: a thread's 16 values are four times four, 128 apart, so that a warp's loads of single values touch neighbouring bytes.
#include <type_traits>

#include "dense8.cuh"

namespace {

// Piece c of a row: its 16 values, or, where rows are not on 16-byte boundaries, the warp's block of 512 dealt four values at a time
template <typename T> __device__ __forceinline__ Piece16<T> load_piece(const T* row, int c, int cols, bool whole) {
    if (whole) return load16(row, c, cols, true);
    T t[16];
    const int at = (c >> 5) * 512 + (c & 31) * 4;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int j = at + (i >> 2) * 128 + (i & 3);
        t[i] = j < cols ? row[j] : narrow<T>(0.f);
    }
    Piece16<T> p;
    memcpy(&p, t, sizeof p);
    return p;
}
__device__ __forceinline__ void store_piece(int8_t* row, int c, int filled, bool whole, const uint4& v) {
    if (whole) {
        if (16 * c < filled) *reinterpret_cast<uint4*>(row + 16 * (size_t)c) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const int at = (c >> 5) * 512 + (c & 31) * 4;
#pragma unroll
    for (int i = 0; i < 4; i++) if (at + i * 128 < filled) *reinterpret_cast<uint32_t*>(row + at + i * 128) = w[i];
}

// grid * (blockDim / (32 group)) rows; group: warps of a row
template <typename T, int KEEP>
__global__ void __launch_bounds__(KEEP == 1 ? 1024 : 512)
quantize_rows_kernel(const T* __restrict__ x, long ldx, int rows, int cols, int whole, int group, int ahead, int8_t* __restrict__ q, long ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[32];
    if (ahead) dep_trigger();
    dep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp / group, step = group * 32, t = threadIdx.x - mine * step, per = (blockDim.x >> 5) / group;
    const int r = blockIdx.x * per + mine, filled = (cols + 127) / 128 * 128, pieces = (filled / 16 + 31) / 32 * 32;
    if (r >= rows) return;                             // (whole groups)
    const T* row = x + (size_t)r * ldx;
    Piece16<T> held[KEEP];
    uint32_t most = 0u;
#pragma unroll
    for (int k = 0; k < KEEP; k++) if (t + k * step < pieces) held[k] = load_piece(row, t + k * step, cols, whole);
#pragma unroll
    for (int k = 0; k < KEEP; k++) if (t + k * step < pieces) most = max(most, most_of(held[k]));
    for (int c = t + KEEP * step; c < pieces; c += step) most = max(most, most_of(load_piece(row, c, cols, whole)));
    most = __reduce_max_sync(0xffffffffu, most);
    if (group > 1) {
        if (lane == 0) red[warp] = most;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + mine), "r"(step) : "memory");
        most = __reduce_max_sync(0xffffffffu, lane < group ? red[mine * group + lane] : 0u);
    }
    const RowScale<T> s(most);
    int8_t* out = q + (size_t)r * ldq;
#pragma unroll
    for (int k = 0; k < KEEP; k++) if (t + k * step < pieces) store_piece(out, t + k * step, filled, whole, s.codes(held[k]));
    for (int c = t + KEEP * step; c < pieces; c += step) store_piece(out, c, filled, whole, s.codes(load_piece(row, c, cols, whole)));
    if (t == 0) scale[r] = s.scale();
    if (!ahead) {
        __threadfence();
        asm volatile("fence.proxy.async.global;" ::: "memory");
    }
}

template <typename T>
int launch_rows(const void* x, long ldx, int rows, int cols, int8_t* q, long ldq, float* scale, int ahead, cudaStream_t st) {
    const int whole = (((uintptr_t)x | ((uintptr_t)ldx * sizeof(T))) & 15) == 0, warps = ((cols + 127) / 128 * 8 + 31) / 32;         // of a thread a piece
    // a CTA a row where they are few, or all resident at once; otherwise as many warps a row as its pieces need, or as give every SM a CTA
    if (rows <= 2 * cmlb_num_sms() || (rows <= 4 * cmlb_num_sms() && (long)rows * warps <= 64l * cmlb_num_sms())) {
        const int group = warps < 32 ? warps : 32;
        CMLB_CUDA(launch_chain(quantize_rows_kernel<T, 1>, dim3(rows), dim3(group * 32), 0, 1, st, static_cast<const T*>(x), ldx, rows, cols, whole, group, ahead, q, ldq, scale));
    } else {
        constexpr int KEEP = 8 / (int)sizeof(T);
        int group = 1;
        while (group < 16 && (group * KEEP < warps || (group < warps && rows * (long)group < 16l * cmlb_num_sms()))) group *= 2;
        CMLB_CUDA(launch_chain(quantize_rows_kernel<T, KEEP>, dim3((rows * (long)group + 15) / 16), dim3(512), 0, 1, st, static_cast<const T*>(x), ldx, rows, cols, whole, group, ahead, q, ldq, scale));
    }
    return CMLB200_OK;
}

}  // namespace

int cmlb_quantize_rows(const void* d_x, int dtype, long ldx, int rows, int cols, int8_t* d_q, long ldq, float* d_scale, int ahead, cudaStream_t st) {
    static const char* who = "cmlb200_quantize_rows";
    CMLB_REQUIRE(d_x && d_q && d_scale && rows > 0, "%s: NULL argument or %d rows", who, rows);
    CMLB_REQUIRE(cols > 0 && cols <= kMaxCols8 && ldx >= cols, "%s: %d columns (up to %d), stride %ld", who, cols, kMaxCols8, ldx);
    CMLB_REQUIRE(ldq % 128 == 0 && ldq >= cols && ((uintptr_t)d_q & 15) == 0, "%s: codes need a stride that is a multiple of 128 (%ld) and 16-byte alignment", who, ldq);
    CMLB_REQUIRE(((uintptr_t)d_scale & 3) == 0 && ((uintptr_t)d_x & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0, "%s: pointers are not aligned to their types", who);
    if (dtype == CMLB200_DT_F32) return launch_rows<float>(d_x, ldx, rows, cols, d_q, ldq, d_scale, ahead, st);
    if (dtype == CMLB200_DT_BF16) return launch_rows<__nv_bfloat16>(d_x, ldx, rows, cols, d_q, ldq, d_scale, ahead, st);
    if (dtype == CMLB200_DT_F16) return launch_rows<__half>(d_x, ldx, rows, cols, d_q, ldq, d_scale, ahead, st);
    CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    return CMLB200_EINVAL;
}

extern "C" int cmlb200_quantize_rows(const void* d_x, int dtype, long ldx, int rows, int cols, int8_t* d_q, long ldq, float* d_scale, void* stream) {
    return cmlb_quantize_rows(d_x, dtype, ldx, rows, cols, d_q, ldq, d_scale, 0, as_stream(stream));
}
