// Attention over 8-bit caches (cache8.cuh), one CTA per row and query head, all arithmetic in fp32: the plainest form.
#include "cache8.cuh"

namespace {

constexpr int A8_THREADS = 128;

__device__ __forceinline__ int first_key8(const cmlb200_attn& a, int p) {
    if (a.chunk > 0) return p / a.chunk * a.chunk;
    return (a.window > 0 && a.window <= p) ? p - a.window + 1 : 0;
}

// grid = (rows, heads), or (tiles * 64, heads) with `tiles`: {first row, rows, slot, position of the first row} each. raw: queries as the projection
// left them, to be normed, given their temperature and turned.
template <bool I8>
__global__ void __launch_bounds__(A8_THREADS)
attention8_rows_kernel(const cmlb200_attn a, const float* __restrict__ qkv, int ld, const int* __restrict__ row_pos, const int* __restrict__ row_slot, const int4* __restrict__ tiles,
                       int raw, __nv_bfloat16* __restrict__ out, int out_ld) {
    extern __shared__ __align__(16) float fs[];
    float* q_s = fs;                                   // [dim]
    float* acc = q_s + a.dim;                          // [vdim]
    __shared__ float sc[A8_THREADS], vw[A8_THREADS], red[32];
    __shared__ int slots[A8_THREADS];
    dep_wait();
    dep_trigger();
    int r = blockIdx.x, p, slot;
    if (tiles) {
        const int4 t = tiles[blockIdx.x >> 6];
        const int i = blockIdx.x & 63;
        if (i >= t.y) return;
        r = t.x + i; p = t.w + i; slot = t.z;
    } else {
        p = row_pos[r]; slot = row_slot[r];
    }
    const int h = blockIdx.y, kh = h / (a.heads / a.kv_heads), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* row = qkv + (size_t)r * ld;
    const int* table = a.block_table + (size_t)slot * a.table_ld;
    const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + (size_t)kh * a.dim_ld;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + (size_t)kh * a.vdim_ld;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float f = 1.0f;
    const float* norm = nullptr;
    if (raw) {
        if (a.q_norm) {
            const int n = a.head_norm ? a.dim : a.heads * a.dim;
            const float* v = a.head_norm ? row + h * a.dim : row;
            f = 1.0f / sqrtf(block_sum(square_share(v, n), red) / (float)n + a.eps);
            norm = a.q_norm + (a.head_norm ? 0 : h * a.dim);
        }
        if (a.temp_every > 0.f) f *= 1.0f + a.temp_coef * logf(floorf((float)(p + 1) / a.temp_every) + 1.0f);
    }
    for (int d = threadIdx.x; d < a.dim; d += A8_THREADS) {
        const float* v = row + h * a.dim;
        float x = v[d] * f * (norm ? norm[d] : 1.0f);
        if (raw && a.freq && d < a.rot_dims) {
            float c, s;
            sincosf((float)p * a.freq[d >> 1], &s, &c);
            const float y = v[d ^ 1] * f * (norm ? norm[d ^ 1] : 1.0f);
            x = (d & 1) ? x * c + y * s : x * c - y * s;
        }
        q_s[d] = x;
    }
    for (int d = threadIdx.x; d < a.vdim; d += A8_THREADS) acc[d] = 0.f;
    auto value = [](const uint8_t* c) {
        if constexpr (I8) return (float)*reinterpret_cast<const int8_t*>(c);
        else { uint32_t lo, hi; unpack8<false>(*c, lo, hi); return half2_floats(lo).x; }
    };
    float m = a.sink ? (a.sinks ? a.sinks[h] : 0.f) : -INFINITY, l = a.sink ? 1.f : 0.f;
    const int k_lo = first_key8(a, p), kept = min(a.keep, k_lo), skip = k_lo - kept, seen = p + 1 - skip;
    auto key_of = [&](int nth) { return nth + (nth < kept ? 0 : skip); };
    for (int kt = 0; kt < seen; kt += A8_THREADS) {
        const int n = min(A8_THREADS, seen - kt);
        __syncthreads();
        if ((int)threadIdx.x < n) {
            const int key = key_of(kt + threadIdx.x);
            slots[threadIdx.x] = table[key / a.block_size] * a.block_size + key % a.block_size;
            vw[threadIdx.x] = a.v_scale[(size_t)(slots[threadIdx.x] / kScaleTokens) * a.kv_heads + kh];
        }
        __syncthreads();
        for (int k = warp; k < n; k += A8_THREADS / 32) {
            const uint8_t* kr = kp + (size_t)slots[k] * a.kv_heads * a.dim_ld;
            float s = 0.f;
            for (int d = lane; d < a.dim; d += 32) s = fmaf(q_s[d], value(kr + d), s);
            s = lane_sum(s);
            if (lane == 0) sc[k] = s * a.k_scale[(size_t)(slots[k] / kScaleTokens) * a.kv_heads + kh] * a.scale - slope * (float)(p - key_of(kt + k));
        }
        __syncthreads();
        float mx = m;
        for (int k = 0; k < n; k++) mx = fmaxf(mx, sc[k]);
        const float c = expf(m - mx);
        m = mx;
        const float w = (int)threadIdx.x < n ? expf(sc[threadIdx.x] - mx) : 0.f;
        l = l * c + block_sum(w, red);
        sc[threadIdx.x] = (int)threadIdx.x < n ? w * vw[threadIdx.x] : 0.f;
        __syncthreads();
        for (int d = threadIdx.x; d < a.vdim; d += A8_THREADS) {
            float x = acc[d] * c;
            for (int k = 0; k < n; k++) x = fmaf(sc[k], value(vp + (size_t)slots[k] * a.kv_heads * a.vdim_ld + d), x);
            acc[d] = x;
        }
    }
    const float inv = (a.out_scale == 0.f ? 1.f : a.out_scale) / l;
    for (int d = threadIdx.x; d < a.vdim; d += A8_THREADS) {
        const float g = a.gate_col < 0 ? 1.0f : sigmoidf(row[a.gate_col + (a.gate_wide ? h * a.vdim + d : h)]);
        out[(size_t)r * out_ld + h * a.vdim + d] = __float2bfloat16_rn(acc[d] * inv * g);
    }
}

int launch(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int rows, const int* d_tiles, int raw, __nv_bfloat16* d_out, int out_ld,
           cudaStream_t st) {
    const size_t smem = sizeof(float) * ((size_t)a->dim + a->vdim);
    const dim3 grid(rows, a->heads);
    if (a->cache_dtype == CMLB200_DT_I8)
        CMLB_CUDA(launch_chain(attention8_rows_kernel<true>, grid, dim3(A8_THREADS), smem, 1, st, *a, d_qkv, ld, d_row_pos, d_row_slot, (const int4*)d_tiles, raw, d_out, out_ld));
    else
        CMLB_CUDA(launch_chain(attention8_rows_kernel<false>, grid, dim3(A8_THREADS), smem, 1, st, *a, d_qkv, ld, d_row_pos, d_row_slot, (const int4*)d_tiles, raw, d_out, out_ld));
    return CMLB200_OK;
}

}  // namespace

int cmlb_attention8_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, cudaStream_t st) {
    return launch(a, d_qkv, ld, nullptr, nullptr, tiles * 64, d_tiles, 0, d_out, out_ld, st);
}
