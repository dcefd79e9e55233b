// Keys and values of projection rows into an 8-bit cache (cache8.cuh): what cmlb200_qk_norm_append and cmlb200_rotate_append do
// for CMLB200_DT_I8 and CMLB200_DT_E4M3.
//
// A scale belongs to 16 tokens, so the rows of a call that fall into one group are one CTA's work, for one key/value head: it takes their
// keys and values through norm and rotation into shared memory, finds the largest of each, settles the scales with those of the group's
// earlier tokens, and writes codes, 16 to a store. Earlier codes are rewritten only where their scale has grown. Bound by the rows' fp32
// columns, which are read once (twice where a norm spans all heads).
#include "cache8.cuh"

namespace {

constexpr int C8_THREADS = 256, C8_WARPS = C8_THREADS / 32;

// grid = (row spans, kv_heads + (queries ? 1 : 0)). A CTA serves the groups whose first row of this call lies in its span.
template <bool I8>
__global__ void __launch_bounds__(C8_THREADS)
cache8_append_kernel(const cmlb200_attn a, float* __restrict__ qkv, int ld, const int* __restrict__ row_pos, const int* __restrict__ row_slot, int first, int rows, int span,
                     int rotate) {
    extern __shared__ __align__(16) float fs[];
    const int dk = a.dim_ld, dv = a.vdim_ld;
    float* ks = fs;                                    // [16][dk]
    float* vs = ks + kScaleTokens * dk;                // [16][dv]
    __shared__ float red_k[C8_WARPS], red_v[C8_WARPS];
    dep_wait();
    dep_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = first + rows;
    const int qw = a.heads * a.dim, kw = a.kv_heads * a.dim, vcol = qw + (a.keys_as_values ? 0 : kw);
    const int lo = first + blockIdx.x * span, hi = min(lo + span, end), h = blockIdx.y;
    const bool turns = rotate && a.freq;
    // a head's entry d of `v` times f * norm, turned with its neighbour
    auto entry = [&](const float* v, const float* norm, float f, int d, int p) {
        float x = v[d] * f * (norm ? norm[d] : 1.0f);
        if (turns && d < a.rot_dims) {
            float c, s;
            sincosf((float)p * a.freq[d >> 1], &s, &c);
            const float y = v[d ^ 1] * f * (norm ? norm[d ^ 1] : 1.0f);
            x = (d & 1) ? x * c + y * s : x * c - y * s;
        }
        return x;
    };
    auto squares = [&](const float* v, int n) {
        float s = 0.f;
        for (int d = lane; d < n; d += 32) s = fmaf(v[d], v[d], s);
        return lane_sum(s);
    };

    if (h == a.kv_heads) {                             // the queries of the span, a warp a row
        for (int r = lo + warp; r < hi; r += C8_WARPS) {
            float* row = qkv + (size_t)r * ld;
            const int p = row_pos[r];
            const float temp = !rotate && a.temp_every > 0.f ? 1.0f + a.temp_coef * logf(floorf((float)(p + 1) / a.temp_every) + 1.0f) : 1.0f;
            float inv = a.q_norm && !a.head_norm ? 1.0f / sqrtf(squares(row, qw) / (float)qw + a.eps) : 1.0f;
            for (int j = 0; j < a.heads; j++) {
                float* v = row + j * a.dim;
                if (a.q_norm && a.head_norm) inv = 1.0f / sqrtf(squares(v, a.dim) / (float)a.dim + a.eps);
                for (int d0 = 0; d0 < a.dim; d0 += 32) {   // (a pair of neighbours lies in one pass of the warp)
                    const int d = d0 + lane;
                    const float x = d < a.dim ? entry(v, a.q_norm ? a.q_norm + (a.head_norm ? 0 : j * a.dim) : nullptr, inv, d, p) * temp : 0.f;
                    __syncwarp();
                    if (d < a.dim) v[d] = x;
                    __syncwarp();
                }
            }
        }
        return;
    }

    for (int r = lo; r < hi;) {
        const int p = row_pos[r], slot = row_slot[r];
        // rows of this group: they follow one another
        auto same = [&](int i) { return row_slot[i] == slot && row_pos[i] - p == i - r && row_pos[i] / kScaleTokens == p / kScaleTokens; };
        int n = 1;
        while (r + n < end && n < kScaleTokens && same(r + n)) n++;
        if (r > first && same(r - 1)) { r += n; continue; }                // begun in front of this span: another CTA's
        const int off = p & (kScaleTokens - 1), page = a.block_table[(size_t)slot * a.table_ld + p / a.block_size], in_page = p & (a.block_size - 1);
        __syncthreads();                               // the previous group's values are written
        for (int i = warp; i < n; i += C8_WARPS) {
            const float* row = qkv + (size_t)(r + i) * ld;
            const float* k = row + qw + h * a.dim;
            float inv = 1.0f;
            if (a.k_norm) {
                const int m = a.head_norm ? a.dim : kw;
                inv = 1.0f / sqrtf(squares(a.head_norm ? k : row + qw, m) / (float)m + a.eps);
            }
            const float* norm = a.k_norm ? a.k_norm + (a.head_norm ? 0 : h * a.dim) : nullptr;
            for (int d = lane; d < dk; d += 32) ks[i * dk + d] = d < a.dim ? cached8(entry(k, norm, inv, d, p + i)) : 0.f;
            const float* v = row + vcol + h * a.vdim;
            for (int d = lane; d < dv; d += 32) vs[i * dv + d] = d < a.vdim ? cached8(v[d]) : 0.f;
        }
        __syncthreads();
        float mk = 0.f, mv = 0.f;
        for (int i = threadIdx.x; i < n * dk; i += C8_THREADS) mk = fmaxf(mk, fabsf(ks[i]));
        for (int i = threadIdx.x; i < n * dv; i += C8_THREADS) mv = fmaxf(mv, fabsf(vs[i]));
        mk = lane_max(mk);
        mv = lane_max(mv);
        if (lane == 0) { red_k[warp] = mk; red_v[warp] = mv; }
        const size_t group = ((size_t)page * (a.block_size / kScaleTokens) + in_page / kScaleTokens) * a.kv_heads + h;
        const float was_k = off ? a.k_scale[group] : 0.f, was_v = off ? a.v_scale[group] : 0.f;
        __syncthreads();                               // (every thread has read the old scales as well)
#pragma unroll
        for (int w = 0; w < C8_WARPS; w++) { mk = fmaxf(mk, red_k[w]); mv = fmaxf(mv, red_v[w]); }
        const float sk = fmaxf(scale8_for<I8>(mk), was_k), sv = fmaxf(scale8_for<I8>(mv), was_v), ik = 1.0f / sk, iv = 1.0f / sv;
        if (threadIdx.x == 0) { a.k_scale[group] = sk; a.v_scale[group] = sv; }
        uint8_t* kd = static_cast<uint8_t*>(a.k_pool) + (((size_t)page * a.block_size + in_page - off) * a.kv_heads + h) * dk;
        uint8_t* vd = static_cast<uint8_t*>(a.v_pool) + (((size_t)page * a.block_size + in_page - off) * a.kv_heads + h) * dv;
        const int kc = dk >> 4, vc = dv >> 4;
        for (int i = threadIdx.x; i < (off + n) * (kc + vc); i += C8_THREADS) {
            const int t = i / (kc + vc), c = i - t * (kc + vc);
            const bool key = c < kc;
            uint4* dst = reinterpret_cast<uint4*>(key ? kd + (size_t)t * a.kv_heads * dk + c * 16 : vd + (size_t)t * a.kv_heads * dv + (c - kc) * 16);
            uint4 u;
            if (t < off) {
                const float was = key ? was_k : was_v, now = key ? sk : sv;
                if (was == now) continue;
                u = *dst;
                const float ratio = was / now;
                u.x = rescale8<I8>(u.x, ratio); u.y = rescale8<I8>(u.y, ratio); u.z = rescale8<I8>(u.z, ratio); u.w = rescale8<I8>(u.w, ratio);
            } else {
                const float* x = key ? ks + (t - off) * dk + c * 16 : vs + (t - off) * dv + (c - kc) * 16;
                const float f = key ? ik : iv;
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = pack8<I8>(x[4 * j] * f, x[4 * j + 1] * f, x[4 * j + 2] * f, x[4 * j + 3] * f);
                u = make_uint4(w[0], w[1], w[2], w[3]);
            }
            *dst = u;
        }
        r += n;
    }
}

}  // namespace

int cmlb_cache8_append(const cmlb200_attn* a, float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int first, int rows, bool rotate, bool queries,
                       cudaStream_t st) {
    const bool q = queries && (a->q_norm || (rotate && a->freq) || (!rotate && a->temp_every > 0.f));
    const int span = rows > 256 ? kScaleTokens : 1;    // a CTA a row while that makes few; then one for the rows that make a whole group
    const dim3 grid((rows + span - 1) / span, a->kv_heads + (q ? 1 : 0));
    const size_t smem = sizeof(float) * kScaleTokens * (size_t)(a->dim_ld + a->vdim_ld);
    CMLB_REQUIRE(smem <= 96 * 1024 && grid.y <= 65535, "8-bit cache: head sizes %d / %d, %d key/value heads", a->dim, a->vdim, a->kv_heads);
    static size_t attr[2][kMaxDevices] = {};
#define C8_LAUNCH(I8)                                                                                                                              \
    do {                                                                                                                                           \
        CMLB_CUDA(cmlb_ensure_smem(cache8_append_kernel<I8>, smem, attr[I8]));                                                                     \
        CMLB_CUDA(launch_chain(cache8_append_kernel<I8>, grid, dim3(C8_THREADS), smem, 1, st, *a, d_qkv, ld, d_row_pos, d_row_slot, first, rows, span, (int)rotate)); \
    } while (0)
    if (a->cache_dtype == CMLB200_DT_I8) C8_LAUNCH(true);
    else C8_LAUNCH(false);
#undef C8_LAUNCH
    return CMLB200_OK;
}
