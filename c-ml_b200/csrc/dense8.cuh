// Rows in 8-bit integers: what quantises them, and what the products over them share.
//
//   a = max(max |x|, 127 2^-126),   scale = a / 127,   code = 127 x / a rounded to the nearest, ties to even
//
// The quotient of a 16-bit number times 127 and a 16-bit number is right to the bit when it is rounded once, ties included, so codes of such rows are those
// of exact arithmetic. It is a product with 127 / a except next to a tie (closer than that product can be off), where it is a division.
#pragma once
#include <type_traits>

#include "lm_util.cuh"

// Where a product's results go, and what makes numbers of its sums
struct Out8 {
    const float *wscale, *bias, *xscale;
    float cap;
    int act, n_out;
    void* y;
    int ldy;
};

// the product of prompt-sized calls (gemm_dense8.cu)
int cmlb_gemm_dense8(const cmlb200_dense8* W, const int8_t* xq, int ldq, int M, const Out8& out, int glu, cudaStream_t st);

namespace {

constexpr int kSkinny8 = 32;                           // rows of x up to which the decode product is taken
constexpr int kMaxCols8 = 131071;                      // 128 * 128 * this is the largest sum that 32 bits hold
constexpr float kLeastMost = 127.f * 1.1754943508222875e-38f;

template <typename T> struct Piece16 { uint4 v[sizeof(T)]; };                // 16 values as they lie (16 bytes hold 16 / sizeof(T) of them)

// value i of a piece of 16-bit or 32-bit floats
template <typename T> __device__ __forceinline__ void widen16(const Piece16<T>& p, float (&x)[16]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else x[i] = __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
    }
}
// magnitude as a whole number: in the order of the magnitudes, infinities above every number and NaN above those
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t most_of(const float (&x)[16]) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, magnitude(x[i]));
    return m;
}

struct RowScale {
    float most, times;                                 // a, 127 / a
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        most = fmaxf(__uint_as_float(bits), kLeastMost);
        times = bits >= 0x7f800000u ? 0.f : __fdiv_rn(127.f, most);
    }
    // a row that holds NaN or an infinity has codes of 0 and scale NaN: whatever is made of it is NaN
    __device__ __forceinline__ bool bad(uint32_t bits) const { return bits >= 0x7f800000u; }
    __device__ __forceinline__ float scale(uint32_t bits) const { return bad(bits) ? __uint_as_float(0x7fffffffu) : __fdiv_rn(most, 127.f); }
    // the code in the low byte
    __device__ __forceinline__ uint32_t code(float x) const {
        const float magic = 12582912.f, r = __fmul_rn(x, times), y = __fadd_rn(r, magic);
        if (fabsf(r - (y - magic)) > 0.5f - 6.1e-5f) {
            const float f = most > 1.2676506e30f ? 2.3283064e-10f : 1.f;       // (127 x stays a number)
            return __float_as_uint(__fadd_rn(__fdiv_rn(__fmul_rn(127.f, x * f), most * f), magic));
        }
        return __float_as_uint(y);
    }
    __device__ __forceinline__ uint4 codes(const float (&x)[16], uint32_t bits) const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = __byte_perm(code(x[4 * i]), code(x[4 * i + 1]), 0x0040), hi = __byte_perm(code(x[4 * i + 2]), code(x[4 * i + 3]), 0x0040);
            w[i] = bad(bits) ? 0u : __byte_perm(lo, hi, 0x5410);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float glu8(int act, float gate, float up) { return unary_act_fast(act, gate) * up; }

// Values 16 c .. 16 c + 15 of a row, zeros behind its end. whole: rows lie on 16-byte boundaries.
template <typename T> __device__ __forceinline__ Piece16<T> load16(const T* row, int c, int cols, bool whole) {
    Piece16<T> p;
    if (whole && 16 * c + 16 <= cols) {
        const uint4* s = reinterpret_cast<const uint4*>(row + 16 * (size_t)c);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) p.v[i] = s[i];
        return p;
    }
    T t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = 16 * c + i < cols ? row[16 * c + i] : narrow<T>(0.f);
    memcpy(&p, t, sizeof p);
    return p;
}

}  // namespace
