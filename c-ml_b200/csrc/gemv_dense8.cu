// Decode products of int8 weights and int8 rows, up to 16 rows of x: y[m][n] = sx[m] sw[n] sum_k xq[m][k] wq[n][k], sums in 32-bit integers, exact; and the entry points of all
// such products.
//
// One CTA an SM, or two, walks over tiles of 16 weight rows (gate and up rows: 32). The weight streams from HBM once, straight into the A fragments of mma.sync m16n8k32: since any order of the
// columns will do as long as both operands use the same one, lane t of a quad takes 16 neighbouring bytes of every 64: one 16-byte load a row feeds two MMAs. The warps split K in
// chunks of 128 columns, each with its next chunks requested RING ahead, across tiles, and the first before the launch waits for its predecessor: weights do not depend on it. Their
// sums meet in shared memory by atomic additions (whole numbers: the order makes no difference).
//
// Rows of x: few of them (M K up to kFused) every CTA quantises itself, into shared memory, while its first weights are on their way: one launch instead of two, and no codes in
// memory. (A warp's work for an output is a few instructions a weight byte, so what bounds these calls is memory, or a launch and its prologue: gate and up rows of 11008x4096 15.7 us for one row of x, 5.7 TB/s;
// 32000x8192 for 4 rows 44 us, 6.0 TB/s; 4096x4096 5.0 us, of which the bytes are 2.6. With CTAs of 16 weight rows each and a launch of its own for the codes: 19.7, 49 and 5.6.)
// More rows come as codes from cmlb200_quantize_rows, through L1, where a warp finds its own columns again with every tile. What is left goes to the tensor-core product of
// prompts (gemm_dense8.cu).
#include <type_traits>

#include "dense8.cuh"

namespace {

__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// RT tiles of 16 weight rows a CTA and turn, NB groups of 8 rows of x. GLU: tile 0 = 16 gate rows, tile 1 = the 16 up rows that go with them. T: what x holds; int8_t: codes
template <typename T, int GW, int RT, int NB, int RING, bool GLU>
__global__ void __launch_bounds__(GW * 32, 16 / GW)
gemv_dense8_kernel(const int8_t* __restrict__ W, int ldw, const T* __restrict__ x, long ldx, int M, int K, int whole, int tiles, const Out8 out) {
    constexpr bool FUSED = sizeof(T) > 1;
    extern __shared__ __align__(16) uint8_t codes_smem[];
    __shared__ int sums[2][RT * 16][NB * 8 + 1];
    __shared__ uint32_t red[GW];
    __shared__ float sxs[NB * 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, chunks = (K + 127) / 128;
    const int lds = chunks * 128 + 64;                 // (rows 64 bytes apart modulo 128: a quarter of a warp reads two of them without a conflict)
    uint4 w[RING][RT][2][2];
    int ftile = warp < chunks ? (int)blockIdx.x : tiles, fc = warp;
    auto fetch = [&](int u) {
        const int8_t* at = W + (size_t)(ftile * (RT * 16) + g) * ldw + fc * 128 + 16 * t;
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    if (ftile < tiles) w[u][i][e][s] = ld_stream(reinterpret_cast<const __nv_bfloat16*>(at + (size_t)(i * 16 + e * 8) * ldw + 64 * s));
        fc += GW;
        if (fc >= chunks) { fc = warp; ftile += gridDim.x; }
    };
#pragma unroll
    for (int u = 0; u < RING; u++) fetch(u);
    for (int i = threadIdx.x; i < 2 * RT * 16 * (NB * 8 + 1); i += GW * 32) (&sums[0][0][0])[i] = 0;
    dep_trigger();
    dep_wait();
    const int8_t* xr[NB];
    if constexpr (FUSED) {
        // a row's warps: 16, 8, 4 or 2
        const int group = M <= 1 ? GW : M <= 2 ? GW / 2 : M <= 4 ? GW / 4 : GW / 8, row = warp / group, step = group * 32, p0 = threadIdx.x - row * step, pieces = chunks * 8;
        constexpr int KEEP = 2;
        const bool on = row < M;
        const T* src = x + (size_t)min(row, M - 1) * ldx;
        Piece16<T> held[KEEP];
        uint32_t most = 0u;
#pragma unroll
        for (int k = 0; k < KEEP; k++) if (on && p0 + k * step < pieces) held[k] = load16(src, p0 + k * step, K, whole);
#pragma unroll
        for (int k = 0; k < KEEP; k++) if (on && p0 + k * step < pieces) most = max(most, most_of(held[k]));
        for (int c = p0 + KEEP * step; on && c < pieces; c += step) most = max(most, most_of(load16(src, c, K, whole)));
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) red[warp] = most;
        __syncthreads();
        most = __reduce_max_sync(0xffffffffu, lane < group ? red[row * group + lane] : 0u);
        const RowScale<T> s(most);
        uint4* dst = reinterpret_cast<uint4*>(codes_smem + (size_t)row * lds);
        if (on) {
#pragma unroll
            for (int k = 0; k < KEEP; k++) if (p0 + k * step < pieces) dst[p0 + k * step] = s.codes(held[k]);
            for (int c = p0 + KEEP * step; c < pieces; c += step) dst[c] = s.codes(load16(src, c, K, whole));
            if (p0 == 0) sxs[row] = s.scale();
        }
        xr[0] = reinterpret_cast<const int8_t*>(codes_smem) + (size_t)min(g, M - 1) * lds + 16 * t;
    } else {
        if ((int)threadIdx.x < M) sxs[threadIdx.x] = out.xscale[threadIdx.x];
#pragma unroll
        for (int b = 0; b < NB; b++) xr[b] = reinterpret_cast<const int8_t*>(x) + (size_t)min(b * 8 + g, M - 1) * ldx + 16 * t;        // rows past M repeat the last, never stored
    }
    __syncthreads();
    int acc[RT][NB][4];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int b = 0; b < NB; b++) acc[i][b][0] = acc[i][b][1] = acc[i][b][2] = acc[i][b][3] = 0;
    int tile = blockIdx.x, c = warp, turn = 0;
    // The warps' sums meet, and 4 NB warps, others every time, finish 16 outputs of NB * 8 rows. Two buffers in turn; who reads a sum leaves 0 for the turn after the next
    auto finish = [&]() {
        int (*mine)[NB * 8 + 1] = sums[turn & 1];
        if (warp < chunks) {
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    atomicAdd(&mine[i * 16 + g][b * 8 + 2 * t], acc[i][b][0]);
                    atomicAdd(&mine[i * 16 + g][b * 8 + 2 * t + 1], acc[i][b][1]);
                    atomicAdd(&mine[i * 16 + g + 8][b * 8 + 2 * t], acc[i][b][2]);
                    atomicAdd(&mine[i * 16 + g + 8][b * 8 + 2 * t + 1], acc[i][b][3]);
                    acc[i][b][0] = acc[i][b][1] = acc[i][b][2] = acc[i][b][3] = 0;
                }
        }
        __syncthreads();
        const int i = ((warp - 4 * NB * turn) & (GW - 1)) * 32 + lane, n = i & 15, m = i >> 4;
        if (m < NB * 8) {
            const int s = mine[n][m], s2 = GLU ? mine[RT * 16 - 16 + n][m] : 0, r = tile * (RT * 16) + n;
            mine[n][m] = 0;
            if (GLU) mine[RT * 16 - 16 + n][m] = 0;
            if (GLU) {
                const int col = tile * 16 + n;
                if (m < M && col < out.n_out)
                    static_cast<__nv_bfloat16*>(out.y)[(size_t)m * out.ldy + col] = __float2bfloat16_rn(glu8(out.act, (float)s * (sxs[m] * out.wscale[r]), (float)s2 * (sxs[m] * out.wscale[r + 16])));
            } else if (m < M && r < out.n_out)
                static_cast<float*>(out.y)[(size_t)m * out.ldy + r] = finish8(s, sxs[m] * out.wscale[r], out.bias ? out.bias[r] : 0.f, out.cap);
        }
        turn++;
        tile += gridDim.x;
        c = warp;
    };
    if (warp >= chunks) {
        while (tile < tiles) finish();
        return;
    }
    while (tile < tiles) {
#pragma unroll
        for (int u = 0; u < RING; u++) {
            if (tile >= tiles) break;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint4 v[NB];
#pragma unroll
                for (int b = 0; b < NB; b++) v[b] = *reinterpret_cast<const uint4*>(xr[b] + (size_t)c * 128 + 64 * s);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        mma_i8(acc[i][b], w[u][i][0][s].x, w[u][i][1][s].x, w[u][i][0][s].y, w[u][i][1][s].y, v[b].x, v[b].y);
                        mma_i8(acc[i][b], w[u][i][0][s].z, w[u][i][1][s].z, w[u][i][0][s].w, w[u][i][1][s].w, v[b].z, v[b].w);
                    }
            }
            fetch(u);
            c += GW;
            if (c >= chunks) finish();
        }
    }
}

// M K up to which the CTAs quantise several rows themselves (a single one always: 8192x28672 41.3 us, two launches 44.2): 4 rows of 4096x4096 5.5 us (two launches 6.2), 8 7.0 (6.4), 2 of 4096x11008 10.6 (11.4), 4 12.3 (11.5)
constexpr int kFused = 24576;
// rows * cols of a weight up to which 9 to 16 rows of x are taken here: 16 of 4096x4096 7.8 us (the prompts' product 8.9), of 11008x4096 14.3 (13.5)
constexpr int kSmall = 20000000;

template <typename T, int GW, int RT, int NB, int RING, bool GLU>
int launch_gemv8(const cmlb200_dense8* W, const void* x, long ldx, int M, const Out8& out, cudaStream_t st) {
    const int whole = (((uintptr_t)x | ((uintptr_t)ldx * sizeof(T))) & 15) == 0, chunks = (W->cols + 127) / 128, tiles = (W->rows + RT * 16 - 1) / (RT * 16);
    const int most = cmlb_num_sms() * (16 / GW);
    const size_t smem = sizeof(T) > 1 ? (size_t)M * (chunks * 128 + 64) : 0;
    static size_t attr[kMaxDevices] = {};
    if (smem) CMLB_CUDA(cmlb_ensure_smem(gemv_dense8_kernel<T, GW, RT, NB, RING, GLU>, smem, attr));
    CMLB_CUDA(launch_chain(gemv_dense8_kernel<T, GW, RT, NB, RING, GLU>, dim3(tiles < most ? tiles : most), dim3(GW * 32), smem, 1, st, static_cast<const int8_t*>(W->w), W->ld,
                           static_cast<const T*>(x), ldx, M, W->cols, whole, tiles, out));
    return CMLB200_OK;
}

size_t codes_bytes(int M, int cols) { return (size_t)M * ((cols + 127) / 128 * 128); }

template <int RT, int RING, bool GLU>
int product8(const cmlb200_dense8* W, const void* x, int dtype, long ldx, int M, Out8 out, void* work, const char* who, cudaStream_t st) {
    if (M == 1 || (M <= 8 && (long)M * W->cols <= kFused)) {
        CMLB_REQUIRE(ldx >= W->cols && ((uintptr_t)x & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0, "%s: %d columns, stride %ld, or x is not aligned to its type", who, W->cols, ldx);
        if (dtype == CMLB200_DT_F32) return launch_gemv8<float, 16, RT, 1, RING, GLU>(W, x, ldx, M, out, st);
        if (dtype == CMLB200_DT_BF16) return launch_gemv8<__nv_bfloat16, 16, RT, 1, RING, GLU>(W, x, ldx, M, out, st);
        if (dtype == CMLB200_DT_F16) return launch_gemv8<__half, 16, RT, 1, RING, GLU>(W, x, ldx, M, out, st);
        CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    }
    int8_t* xq = static_cast<int8_t*>(work);
    const int ldq = (W->cols + 127) / 128 * 128;
    float* xs = reinterpret_cast<float*>(xq + codes_bytes(M, W->cols));
    const int rc = cmlb_quantize_rows(x, dtype, ldx, M, W->cols, xq, ldq, xs, 1, st);
    if (rc) return rc;
    out.xscale = xs;
    if (M <= 8 || (M <= 16 && (long)W->rows * W->cols <= kSmall)) {
        constexpr int G = GLU ? 16 : 8;                // (two CTAs an SM take tiles of 16 weight rows beside one another: 8 rows of 4096x4096 6.95 to 6.4 us, gate and up rows 19.0 and 20.4)
        return M <= 8 ? launch_gemv8<int8_t, G, RT, 1, RING, GLU>(W, xq, ldq, M, out, st) : launch_gemv8<int8_t, G, RT, 2, RING, GLU>(W, xq, ldq, M, out, st);
    }
    return cmlb_gemm_dense8(W, xq, ldq, M, out, GLU, st);
}

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
    return codes_bytes(M, cols) + ((size_t)M * 4 + 15) / 16 * 16;
}

extern "C" int cmlb200_linear_dense8(const cmlb200_dense8* W, const void* d_x, int dtype, long ldx, int M, float* d_y, long ldy, void* d_work, void* stream) {
    static const char* who = "cmlb200_linear_dense8";
    int rc = check8(W, d_x, M, d_y, d_work, who);
    if (rc) return rc;
    CMLB_REQUIRE(ldy >= W->rows && ((uintptr_t)d_y & 3) == 0, "%s: output stride %ld", who, ldy);
    const Out8 out = {W->scale, W->bias, nullptr, W->cap, 0, W->rows, d_y, ldy};
    return product8<1, 4, false>(W, d_x, dtype, ldx, M, out, d_work, who, as_stream(stream));
}

extern "C" int cmlb200_linear_dense8_glu(const cmlb200_dense8* W, const void* d_x, int dtype, long ldx, int M, int ff, int act, uint16_t* d_f, long ldf, void* d_work, void* stream) {
    static const char* who = "cmlb200_linear_dense8_glu";
    int rc = check8(W, d_x, M, d_f, d_work, who);
    if (rc) return rc;
    CMLB_REQUIRE(ff > 0 && W->rows == 2 * ((ff + 15) & ~15) && ldf >= ff && ((uintptr_t)d_f & 1) == 0, "%s: %d weight rows for %d outputs, stride %ld", who, W->rows, ff, ldf);
    CMLB_REQUIRE(act == CMLB200_ACT_SILU || act == CMLB200_ACT_GELU_TANH || act == CMLB200_ACT_GELU_ERF, "%s: activation %d", who, act);
    const Out8 out = {W->scale, nullptr, nullptr, 0.f, act, ff, d_f, ldf};
    return product8<2, 2, true>(W, d_x, dtype, ldx, M, out, d_work, who, as_stream(stream));
}
