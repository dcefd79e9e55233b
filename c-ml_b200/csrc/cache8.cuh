// Pieces of the kernels over 8-bit key/value caches (cache_dtype CMLB200_DT_I8 and CMLB200_DT_E4M3): a pool holds codes, and every
// group of 16 tokens of a page has a scale per key/value head. A value is code * scale.
//
// A scale is the smallest power of two, at least 2^-126, whose 127 (int8) or 448 (e4m3) multiples hold the largest value of the group.
// Dividing by it is exact, so a code is the value's one rounding, and codes that a later, larger token makes too fine are halved, quartered
// and so on: a value that was rounded at several scales on the way is off by half a step of each, less than one step of the last.
#pragma once
#include <cuda_fp8.h>
#include "lm_util.cuh"

namespace {

constexpr int kScaleTokens = 16;

// The first key that the row at position p sees, the kept ones (0 .. keep - 1) aside.
__device__ __forceinline__ int first_key8(const cmlb200_attn& a, int p) {
    if (a.chunk > 0) return p / a.chunk * a.chunk;
    return (a.window > 0 && a.window <= p) ? p - a.window + 1 : 0;
}

// The smallest allowed power of two that holds `most` (not negative, at most 65504).
template <bool I8> __device__ __forceinline__ float scale8_for(float most) {
    // most = m 2^x with 1/2 <= m < 1; 127 = 127/128 2^7, 448 = 7/8 2^9
    constexpr int fits = I8 ? 7 : 9;
    constexpr uint32_t edge = I8 ? 0x7E0000u : 0x600000u;
    const uint32_t b = __float_as_uint(most);
    const int x = (int)(b >> 23) - 126;
    return __uint_as_float((uint32_t)(max(x - fits + ((b & 0x7FFFFFu) > edge), -126) + 127) << 23);
}
// what enters the cache: numbers beyond fp16's range are held at its end, as in fp16 caches; NaN is zero
__device__ __forceinline__ float cached8(float v) { return v != v ? 0.f : fminf(fmaxf(v, -65504.f), 65504.f); }

// four codes, the first in the lowest byte; values are in units of the scale
template <bool I8> __device__ __forceinline__ uint32_t pack8(float a, float b, float c, float d) {
    if constexpr (I8) {
        const uint32_t lo = __byte_perm((uint32_t)__float2int_rn(a), (uint32_t)__float2int_rn(b), 0x0040);
        const uint32_t hi = __byte_perm((uint32_t)__float2int_rn(c), (uint32_t)__float2int_rn(d), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    } else {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
}
// The values of the two lower and the two upper codes of a word, exact in fp16. int8: a code plus 128 is the low byte of the fp16
// number 1024 + code + 128.
template <bool I8> __device__ __forceinline__ void unpack8(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (I8) {
        const uint32_t u = w ^ 0x80808080u, base = 0x64806480u;        // 1152
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(base));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(base));
    } else {
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(w));
    }
}
__device__ __forceinline__ float2 half2_floats(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// A word's codes for a scale that has grown: `ratio`, the old scale over the new one, is a power of two.
template <bool I8> __device__ __forceinline__ uint32_t rescale8(uint32_t w, float ratio) {
    uint32_t lo, hi;
    unpack8<I8>(w, lo, hi);
    const float2 a = half2_floats(lo), b = half2_floats(hi);
    return pack8<I8>(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

// Clusters of k CTAs of a kernel that run at a time; -1: none.
inline int cluster_room(const void* kern, int k, int threads, size_t smem) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)k;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(k);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n > 0) return n;
    cudaGetLastError();
    return k == 1 ? cmlb_num_sms() : -1;
}

__host__ __device__ inline bool is_cache8(int dtype) { return dtype == CMLB200_DT_I8 || dtype == CMLB200_DT_E4M3; }

}  // namespace

// Appends rows first .. first + rows - 1 to an 8-bit cache (cache8_append.cu). queries: the rows' queries are normed (and turned, with
// `rotate`) in place as well; otherwise the rows are only read.
int cmlb_cache8_append(const cmlb200_attn* a, float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int first, int rows, bool rotate, bool queries,
                       cudaStream_t st);
// the current device's word of cmlb200_attention8_status
int cmlb_attention8_status_word(int** word);
int cmlb_attention8_one(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int rows, int max_keys, __nv_bfloat16* d_out, int out_ld,
                        cudaStream_t st);
int cmlb_attention8_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, cudaStream_t st);
