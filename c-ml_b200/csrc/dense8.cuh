// Rows in 8-bit integers: what quantises them, and what the products over them share.
//
//   a = max(max |x|, 127 2^-126),   scale = a / 127,   code = 127 x / a rounded to the nearest, ties to even
//
// The quotient is a product with 127 / a, except next to a tie (closer than that product can be off), where the sign of 127 x - (k + 1/2) a decides. 127 times a number of 16 bits is exact, so
// codes of such rows are those of exact arithmetic, ties included. Where a's odd part is not a multiple of 127, which is prime, such numbers have no ties but 127 x / a = 63.5, half the
// largest, and come no closer to one than 2^-20 of themselves: 127 / a a little (2^-22) larger gives every code, and nothing has to be looked at.
#pragma once
#include <type_traits>

#include "lm_util.cuh"
#include "pairs.cuh"

// Where a product's results go, and what makes numbers of its sums
struct Out8 {
    const float *wscale, *bias, *xscale;
    float cap;
    int act, n_out;
    void* y;
    long ldy;
};

// cmlb200_quantize_rows; ahead: launches behind it begin before it has written anything (quantize_rows.cu)
int cmlb_quantize_rows(const void* d_x, int dtype, long ldx, int rows, int cols, int8_t* d_q, long ldq, float* d_scale, int ahead, cudaStream_t st);
// the product of prompt-sized calls (gemm_dense8.cu)
int cmlb_gemm_dense8(const cmlb200_dense8* W, const int8_t* xq, int ldq, int M, const Out8& out, int glu, cudaStream_t st);

namespace {

constexpr int kMaxCols8 = 131071;                      // 128 * 128 * this is the largest sum that 32 bits hold
constexpr float kLeastMost = 127.f * 1.1754943508222875e-38f;

template <typename T> struct Piece16 { uint4 v[sizeof(T)]; };                // 16 values as they lie (16 bytes hold 16 / sizeof(T) of them)

// value i of a piece of 16-bit or 32-bit floats
template <typename T> __device__ __forceinline__ float value16(const Piece16<T>& p, int i) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
}
// The largest magnitude of a piece as a whole number: in the order of the magnitudes, infinities above every number and NaN above those. 16-bit values two at a time
template <typename T> __device__ __forceinline__ uint32_t most_of(const Piece16<T>& p) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
    if constexpr (sizeof(T) == 4) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 16; i++) m = max(m, w[i] & 0x7fffffffu);
        return m;
    } else {
        typedef std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162> T2;
        T2 m, t;
        memcpy(&m, &w[0], 4);
        m = __habs2(m);
#pragma unroll
        for (int i = 1; i < 8; i++) {
            memcpy(&t, &w[i], 4);
            m = __hmax2_nan(m, __habs2(t));
        }
        return max(__float_as_uint(widen(m.x)) & 0x7fffffffu, __float_as_uint(widen(m.y)) & 0x7fffffffu);
    }
}

constexpr float kMagic = 12582912.f;                   // a number added to it is rounded to a whole one, in its low bits
constexpr float kNear = 2.3841858e-7f;                 // 2^-22: four times what 127 / a is off by
// Next to a tie h: 127 x - h a has the right sign, and is 0 for a tie alone, since it is rounded once
__device__ __forceinline__ uint32_t settle(float x, float times, float most, float unit) {
    const float r = __fmul_rn(x, times), k = __fadd_rn(r, kMagic) - kMagic;
    float whole = k;
    if (fabsf(r - k) > 0.4375f) {
        const float h = k + copysignf(0.5f, r - k), d = fmaf(-h, most, __fmul_rn(127.f, x * unit));
        whole = d == 0.f ? h : h + copysignf(0.5f, d);
    }
    return __float_as_uint(whole + kMagic) & 0xffu;
}
// not inlined: the kernels' code stays small, which matters where it is fetched anew with every launch
__device__ __noinline__ uint32_t settled_codes(float4 x, float times, float most, float unit) {
    return settle(x.x, times, most, unit) | settle(x.y, times, most, unit) << 8 | settle(x.z, times, most, unit) << 16 | settle(x.w, times, most, unit) << 24;
}

template <typename T> struct RowScale {
    float most, times, unit;                           // a, what numbers are multiplied with, a power of two that keeps 127 x and a within range
    bool bad, sure;                                    // a row that holds NaN or an infinity has codes of 0 and scale NaN: whatever is made of it is NaN; a product decides every code
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        bad = bits >= 0x7f800000u;
        most = fmaxf(__uint_as_float(bits), kLeastMost);
        times = __fdiv_rn(127.f, most);
        unit = most > 1.2676506e30f ? 2.3283064e-10f : most < 8.6736174e-19f ? 1.8446744e19f : 1.f;
        sure = false;
        if (sizeof(T) == 2) {
            const uint32_t m = (__float_as_uint(most) & 0x7fffffu) | 0x800000u, odd = m >> (__ffs(m) - 1);
            sure = odd == 127u || odd % 127u != 0u;    // (odd = 127: 127 / a is a power of two)
            if (odd % 127u != 0u) times *= 1.f + kNear;
        }
    }
    __device__ __forceinline__ float scale() const { return bad ? __uint_as_float(0x7fffffffu) : __fdiv_rn(most, 127.f); }
    static __device__ __forceinline__ uint32_t bytes(uint64_t y01, uint64_t y23) {
        return __byte_perm(__byte_perm((uint32_t)y01, (uint32_t)(y01 >> 32), 0x0040), __byte_perm((uint32_t)y23, (uint32_t)(y23 >> 32), 0x0040), 0x5410);
    }
    // Four codes in a word, two values an instruction. Not sure: of products with a little less and a little more than 127 / a, which agree except next to a tie
    __device__ __forceinline__ uint32_t codes(float x0, float x1, float x2, float x3) const {
        const uint64_t a = pair_of(x0, x1), b = pair_of(x2, x3), magic = pair_of(kMagic, kMagic);
        if (sizeof(T) == 2 && sure) {
            const uint64_t f = pair_of(times, times);
            return bytes(fma_pair(a, f, magic), fma_pair(b, f, magic));
        }
        const uint64_t lo = pair_of(times * (1.f - kNear), times * (1.f - kNear)), hi = pair_of(times * (1.f + kNear), times * (1.f + kNear));
        const uint32_t w = bytes(fma_pair(a, lo, magic), fma_pair(b, lo, magic)), v = bytes(fma_pair(a, hi, magic), fma_pair(b, hi, magic));
        return w == v ? w : settled_codes(make_float4(x0, x1, x2, x3), times, most * unit, unit);
    }
    __device__ __forceinline__ uint4 codes(const Piece16<T>& p) const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = codes(value16(p, 4 * i), value16(p, 4 * i + 1), value16(p, 4 * i + 2), value16(p, 4 * i + 3));
            if (bad) w[i] = 0u;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// A result from its sum: the scales' product is rounded, then the sum with the bias as one; the same in all kernels, so that a row's results do not depend on how many rows there are
__device__ __noinline__ float far_cap(float y, float cap) { return soft_cap(y, cap); }          // (out of the way)
__device__ __forceinline__ float finish8(int sum, float unit, float bias, float cap) {
    const float y = fmaf((float)sum, unit, bias);
    return cap > 0.f ? far_cap(y, cap) : y;
}
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
