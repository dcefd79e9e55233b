// Decode product of int8 weights and int8 rows, up to 32 rows of x a pass: y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k], sums in 32-bit integers, exact.
// The weight streams from HBM once, straight into the A fragments of mma.sync m16n8k32: since any order of the columns will do as long as both operands
// use the same one, lane t of a quad takes 16 neighbouring bytes of every 64: one 16-byte load a row feeds two MMAs. Codes of x come the same way through L1.
// The warps of a CTA split K and meet in shared memory; whole numbers, so in any order.
//
// The first weights are requested before the launch waits for its predecessor: they do not depend on it.
#include <type_traits>

#include "dense8.cuh"

namespace {

constexpr int GW = 8;                                  // warps

__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// RT tiles of 16 weight rows per CTA, NB groups of 8 rows of x; blockIdx.y: passes of NB * 8 rows. GLU: tile 0 = 16 gate rows, tile 1 = the 16 up rows that go with them.
template <int RT, int NB, bool GLU>
__global__ void __launch_bounds__(GW * 32)
gemv_dense8_kernel(const int8_t* __restrict__ W, int ldw, const int8_t* __restrict__ xq, int ldx, int M, int K, const Out8 out) {
    __shared__ int part[GW][RT * 16][NB * 8 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * RT * 16, chunks = (K + 127) / 128, m0 = blockIdx.y * NB * 8;
    const int8_t* wrow[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        wrow[i][0] = W + (size_t)(n0 + i * 16 + g) * ldw + 16 * t;
        wrow[i][1] = wrow[i][0] + (size_t)8 * ldw;
    }
    constexpr int RING = 4 / RT;                       // 128-column chunks in flight per warp
    uint4 w[RING][RT][2][2];
    auto fetch = [&](int u, int c) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    w[u][i][e][s] = c < chunks ? ld_stream(reinterpret_cast<const __nv_bfloat16*>(wrow[i][e] + (size_t)c * 128 + 64 * s)) : make_uint4(0u, 0u, 0u, 0u);
    };
#pragma unroll
    for (int u = 0; u < RING; u++) fetch(u, warp + u * GW);
    dep_trigger();
    dep_wait();
    int acc[RT][NB][4];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int b = 0; b < NB; b++) acc[i][b][0] = acc[i][b][1] = acc[i][b][2] = acc[i][b][3] = 0;
    const int8_t* xr[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) xr[b] = xq + (size_t)min(m0 + b * 8 + g, M - 1) * ldx + 16 * t;       // rows past M repeat the last, never stored
    for (int c0 = warp; c0 < chunks; c0 += RING * GW) {
#pragma unroll
        for (int u = 0; u < RING; u++) {
            const int c = min(c0 + u * GW, chunks - 1);              // past the end: zero weights
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(xr[b] + (size_t)c * 128 + 64 * s);
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        mma_i8(acc[i][b], w[u][i][0][s].x, w[u][i][1][s].x, w[u][i][0][s].y, w[u][i][1][s].y, v.x, v.y);
                        mma_i8(acc[i][b], w[u][i][0][s].z, w[u][i][1][s].z, w[u][i][0][s].w, w[u][i][1][s].w, v.z, v.w);
                    }
                }
            fetch(u, c0 + (u + RING) * GW);
        }
    }
    // accumulator 0, 1: weight row g, rows 2t, 2t + 1 of x; 2, 3: weight row g + 8
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            part[warp][i * 16 + g][b * 8 + 2 * t] = acc[i][b][0];
            part[warp][i * 16 + g][b * 8 + 2 * t + 1] = acc[i][b][1];
            part[warp][i * 16 + g + 8][b * 8 + 2 * t] = acc[i][b][2];
            part[warp][i * 16 + g + 8][b * 8 + 2 * t + 1] = acc[i][b][3];
        }
    __syncthreads();
    constexpr int OUT = GLU ? 16 : RT * 16;
    for (int i = threadIdx.x; i < OUT * NB * 8; i += GW * 32) {
        const int n = i % OUT, m = i / OUT;
        if (m0 + m >= M) break;
        int s = 0, s2 = 0;
#pragma unroll
        for (int k = 0; k < GW; k++) {
            s += part[k][n][m];
            if (GLU) s2 += part[k][RT * 16 - 16 + n][m];
        }
        const float sx = out.xscale[m0 + m];
        if (GLU) {
            const int c = blockIdx.x * 16 + n;
            if (c < out.n_out)
                static_cast<__nv_bfloat16*>(out.y)[(size_t)(m0 + m) * out.ldy + c] = __float2bfloat16_rn(
                    glu8(out.act, (float)s * (sx * out.wscale[n0 + n]), (float)s2 * (sx * out.wscale[n0 + 16 + n])));
        } else if (n0 + n < out.n_out) {
            float y = (float)s * (sx * out.wscale[n0 + n]);
            if (out.bias) y += out.bias[n0 + n];
            if (out.cap > 0.f) y = soft_cap(y, out.cap);
            static_cast<float*>(out.y)[(size_t)(m0 + m) * out.ldy + n0 + n] = y;
        }
    }
}

template <int RT, bool GLU>
int launch_gemv8(const cmlb200_dense8* W, const int8_t* xq, int ldx, int M, const Out8& out, cudaStream_t st) {
    const unsigned tiles = (unsigned)((W->rows + RT * 16 - 1) / (RT * 16));
#define G8_LAUNCH(NB) CMLB_CUDA(launch_chain(gemv_dense8_kernel<RT, NB, GLU>, dim3(tiles, (unsigned)((M + NB * 8 - 1) / (NB * 8))), dim3(GW * 32), 0, 1, st, static_cast<const int8_t*>(W->w), W->ld, xq, ldx, M, W->cols, out))
    if (M <= 8) G8_LAUNCH(1);
    else if (M <= 16) G8_LAUNCH(2);
    else G8_LAUNCH(4);
#undef G8_LAUNCH
    return CMLB200_OK;
}

size_t codes_bytes(int M, int cols) { return (size_t)M * ((cols + 127) / 128 * 128); }

int check8(const cmlb200_dense8* W, const void* x, int M, void* y, void* work, const char* who) {
    CMLB_REQUIRE(W && W->w && W->scale && x && y && work, "%s: NULL argument", who);
    CMLB_REQUIRE(W->rows > 0 && W->cols > 0 && W->cols <= kMaxCols8 && W->ld % 128 == 0 && W->ld >= W->cols, "%s: bad weight [%d, %d], stride %d", who, W->rows, W->cols, W->ld);
    CMLB_REQUIRE(M > 0 && M <= (1 << 20), "%s: %d rows", who, M);
    CMLB_REQUIRE((((uintptr_t)W->w | (uintptr_t)work) & 15) == 0 && (((uintptr_t)W->scale | (uintptr_t)W->bias) & 3) == 0, "%s: weight and workspace need 16-byte alignment", who);
    return CMLB200_OK;
}

}  // namespace

extern "C" size_t cmlb200_dense8_work_bytes(int M, int rows, int cols) {
    if (M <= 0 || rows <= 0 || cols <= 0) return 0;
    return codes_bytes(M, cols) + ((size_t)M + 275) / 4 * 16;      // (the prompts' kernel reads scales of whole tiles)
}

extern "C" int cmlb200_linear_dense8(const cmlb200_dense8* W, const void* d_x, int dtype, long ldx, int M, float* d_y, long ldy, void* d_work, void* stream) {
    static const char* who = "cmlb200_linear_dense8";
    int rc = check8(W, d_x, M, d_y, d_work, who);
    if (rc) return rc;
    CMLB_REQUIRE(ldy >= W->rows && ((uintptr_t)d_y & 3) == 0, "%s: output stride %ld", who, ldy);
    int8_t* xq = static_cast<int8_t*>(d_work);
    const int ldq = (W->cols + 127) / 128 * 128;
    float* xs = reinterpret_cast<float*>(xq + codes_bytes(M, W->cols));
    rc = cmlb200_quantize_rows(d_x, dtype, ldx, M, W->cols, xq, ldq, xs, stream);
    if (rc) return rc;
    const Out8 out = {W->scale, W->bias, xs, W->cap, 0, W->rows, d_y, (int)ldy};
    return M <= kSkinny8 ? launch_gemv8<1, false>(W, xq, ldq, M, out, as_stream(stream)) : cmlb_gemm_dense8(W, xq, ldq, M, out, 0, as_stream(stream));
}

extern "C" int cmlb200_linear_dense8_glu(const cmlb200_dense8* W, const void* d_x, int dtype, long ldx, int M, int ff, int act, uint16_t* d_f, long ldf, void* d_work, void* stream) {
    static const char* who = "cmlb200_linear_dense8_glu";
    int rc = check8(W, d_x, M, d_f, d_work, who);
    if (rc) return rc;
    CMLB_REQUIRE(ff > 0 && W->rows == 2 * ((ff + 15) & ~15) && ldf >= ff && ((uintptr_t)d_f & 1) == 0, "%s: %d weight rows for %d outputs, stride %ld", who, W->rows, ff, ldf);
    CMLB_REQUIRE(act == CMLB200_ACT_SILU || act == CMLB200_ACT_GELU_TANH || act == CMLB200_ACT_GELU_ERF, "%s: activation %d", who, act);
    int8_t* xq = static_cast<int8_t*>(d_work);
    const int ldq = (W->cols + 127) / 128 * 128;
    float* xs = reinterpret_cast<float*>(xq + codes_bytes(M, W->cols));
    rc = cmlb200_quantize_rows(d_x, dtype, ldx, M, W->cols, xq, ldq, xs, stream);
    if (rc) return rc;
    const Out8 out = {W->scale, nullptr, xs, 0.f, act, ff, d_f, (int)ldf};
    return M <= kSkinny8 ? launch_gemv8<2, true>(W, xq, ldq, M, out, as_stream(stream)) : cmlb_gemm_dense8(W, xq, ldq, M, out, 1, as_stream(stream));
}
