// Keys and values of projection rows into an 8-bit cache (cache8.cuh): what cmlb200_qk_norm_append and cmlb200_rotate_append do
// for CMLB200_DT_I8 and CMLB200_DT_E4M3.
//
// A scale belongs to 16 tokens, so the rows of a call that fall into one group are one CTA's work, for one key/value head. A warp takes two of the
// rows, a lane four neighbouring dimensions of each (and of the 128 behind, where heads are that wide): norm and rotation stay in the lane, the largest
// magnitudes meet in shared memory once, the scales are settled with those of the group's earlier tokens, and a lane's four codes are one store of a
// row's contiguous ones. Earlier codes are rewritten only where their scale has grown. Everything a CTA needs is requested before its first wait.
// Bound by the rows' fp32 columns, which are read once (the keys again where a norm spans all heads), and by how little of it is under way: a CTA serves one group, so 4,096 rows
// of 8 heads of 128 take three and a half rounds of positions, rows, page and scale, and nothing of the next group is requested meanwhile: 12.7 us (42 MB, 3.3 TB/s; e4m3 13.2), 64 rows
// in 3.4, most of it a launch and two dependent loads. Queries that are normed or turned are rewritten by one CTA for 16 rows: 4,096 rows of 32 query heads 72 us, 512 25 to 32. (With a loop over the rows' positions in place of the one ballot that finds a group's rows: 48.8 and 11.3 us.)
#include "cache8.cuh"

namespace {

constexpr int C8_THREADS = 256, C8_WARPS = C8_THREADS / 32, C8_ROWS = kScaleTokens / C8_WARPS;

// entries d .. d + 3 of n; zeros behind them
__device__ __forceinline__ float4 four_of(const float* v, int d, int n, bool vec) {
    if (vec) return d < n ? *reinterpret_cast<const float4*>(v + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(d < n ? v[d] : 0.f, d + 1 < n ? v[d + 1] : 0.f, d + 2 < n ? v[d + 2] : 0.f, d + 3 < n ? v[d + 3] : 0.f);
}
__device__ __forceinline__ float largest(const float4& v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }
// entries d .. d + 3 of a head at position p, turned
__device__ __forceinline__ void turn_four(const cmlb200_attn& a, float4& v, int d, int p) {
    float c, s;
    if (d < a.rot_dims) {
        sincosf((float)p * a.freq[d >> 1], &s, &c);
        v = make_float4(v.x * c - v.y * s, v.y * c + v.x * s, v.z, v.w);
    }
    if (d + 2 < a.rot_dims) {
        sincosf((float)p * a.freq[(d >> 1) + 1], &s, &c);
        v = make_float4(v.x, v.y, v.z * c - v.w * s, v.w * c + v.z * s);
    }
}
template <int N> __device__ __forceinline__ float squares(const float4 (&x)[N]) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) s = fmaf(x[j].x, x[j].x, fmaf(x[j].y, x[j].y, fmaf(x[j].z, x[j].z, fmaf(x[j].w, x[j].w, s))));
    return lane_sum(s);
}
template <int N> __device__ __forceinline__ void times(float4 (&x)[N], float f, const float* norm, int n, int lane) {
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float4 w = norm ? four_of(norm, 4 * lane + 128 * j, n, false) : make_float4(1.f, 1.f, 1.f, 1.f);
        x[j] = make_float4(x[j].x * f * w.x, x[j].y * f * w.y, x[j].z * f * w.z, x[j].w * f * w.w);
    }
}

// grid = (row spans, kv_heads + (queries ? 1 : 0)). A CTA serves the groups whose first row of this call lies in its span. N: lanes' shares of a head, 128 dimensions
// together. VEC: heads and rows begin on 16-byte boundaries.
template <bool I8, int N, bool VEC>
__global__ void __launch_bounds__(C8_THREADS)
cache8_append_kernel(const cmlb200_attn a, float* __restrict__ qkv, int ld, const int* __restrict__ row_pos, const int* __restrict__ row_slot, int first, int rows, int span,
                     int rotate) {
    __shared__ float red_k[C8_WARPS], red_v[C8_WARPS], red[32];
    dep_wait();
    dep_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = first + rows;
    const int qw = a.heads * a.dim, kw = a.kv_heads * a.dim, vcol = qw + (a.keys_as_values ? 0 : kw);
    const int lo = first + blockIdx.x * span, hi = min(lo + span, end), h = blockIdx.y;
    const bool turns = rotate && a.freq;

    if (h == a.kv_heads) {                             // the queries of the span, row by row, a warp a head
        for (int r = lo; r < hi; r++) {
            const int p = row_pos[r];
            float* row = qkv + (size_t)r * ld;
            const float temp = !rotate && a.temp_every > 0.f ? 1.0f + a.temp_coef * logf(floorf((float)(p + 1) / a.temp_every) + 1.0f) : 1.0f;
            const bool whole = a.q_norm && !a.head_norm;
            const float inv = whole ? 1.0f / sqrtf(block_sum(square_share(row, qw), red) / (float)qw + a.eps) : 1.0f;      // (behind it all have read the row)
            for (int j = warp; j < a.heads; j += C8_WARPS) {
                float* v = row + j * a.dim;
                float4 x[N];
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = four_of(v, 4 * lane + 128 * i, a.dim, VEC);
                const float f = a.q_norm && a.head_norm ? 1.0f / sqrtf(squares(x) / (float)a.dim + a.eps) : inv;
                times(x, f * temp, a.q_norm ? a.q_norm + (whole ? j * a.dim : 0) : nullptr, a.dim, lane);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int d = 4 * lane + 128 * i;
                    if (turns) turn_four(a, x[i], d, p);
                    if (VEC) {
                        if (d < a.dim) *reinterpret_cast<float4*>(v + d) = x[i];
                    } else {
                        if (d < a.dim) v[d] = x[i].x;
                        if (d + 1 < a.dim) v[d + 1] = x[i].y;
                        if (d + 2 < a.dim) v[d + 2] = x[i].z;
                        if (d + 3 < a.dim) v[d + 3] = x[i].w;
                    }
                }
            }
        }
        return;
    }

    for (int r = lo; r < hi;) {
        // lane l looks at row r - 1 + l: the rows of this group follow one another
        const int at = r - 1 + lane, q = min(max(at, first), end - 1), its_pos = row_pos[q], its_slot = row_slot[q];
        const int p = __shfl_sync(0xffffffffu, its_pos, 1), slot = __shfl_sync(0xffffffffu, its_slot, 1);
        const unsigned same = __ballot_sync(0xffffffffu, at >= first && at < end && its_slot == slot && its_pos - p == at - r && its_pos / kScaleTokens == p / kScaleTokens);
        const int n = min(kScaleTokens, __ffs(~(same >> 1)) - 1);
        if (same & 1) { r += n; continue; }            // begun in front of this span: another CTA's
        float4 k[C8_ROWS][N], v[C8_ROWS][N];
#pragma unroll
        for (int i = 0; i < C8_ROWS; i++) {
            const int j = warp + i * C8_WARPS;
            const float* row = qkv + (size_t)(r + min(j, n - 1)) * ld;
#pragma unroll
            for (int e = 0; e < N; e++) {
                k[i][e] = four_of(row + qw + h * a.dim, 4 * lane + 128 * e, a.dim, VEC);
                v[i][e] = four_of(row + vcol + h * a.vdim, 4 * lane + 128 * e, a.vdim, VEC);
            }
        }
        const int off = p & (kScaleTokens - 1), page = a.block_table[(size_t)slot * a.table_ld + p / a.block_size], in_page = p & (a.block_size - 1);
        const size_t group = ((size_t)page * (a.block_size / kScaleTokens) + in_page / kScaleTokens) * a.kv_heads + h;
        const float was_k = off ? a.k_scale[group] : 0.f, was_v = off ? a.v_scale[group] : 0.f;
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int i = 0; i < C8_ROWS; i++) {
            const int j = warp + i * C8_WARPS;
            if (j >= n) continue;                      // (the same for a whole warp)
            if (a.k_norm) {
                const float* whole = qkv + (size_t)(r + j) * ld + qw;
                float ss = 0.f;
                if (!a.head_norm) for (int d = lane; d < kw; d += 32) ss = fmaf(whole[d], whole[d], ss);
                ss = a.head_norm ? squares(k[i]) : lane_sum(ss);
                times(k[i], 1.0f / sqrtf(ss / (float)(a.head_norm ? a.dim : kw) + a.eps), a.k_norm + (a.head_norm ? 0 : h * a.dim), a.dim, lane);
            }
#pragma unroll
            for (int e = 0; e < N; e++) {
                if (turns) turn_four(a, k[i][e], 4 * lane + 128 * e, p + j);
                k[i][e] = make_float4(cached8(k[i][e].x), cached8(k[i][e].y), cached8(k[i][e].z), cached8(k[i][e].w));
                v[i][e] = make_float4(cached8(v[i][e].x), cached8(v[i][e].y), cached8(v[i][e].z), cached8(v[i][e].w));
                mk = fmaxf(mk, largest(k[i][e]));
                mv = fmaxf(mv, largest(v[i][e]));
            }
        }
        mk = lane_max(mk);
        mv = lane_max(mv);
        __syncthreads();                               // the previous group's maxima have been read
        if (lane == 0) { red_k[warp] = mk; red_v[warp] = mv; }
        __syncthreads();                               // (every thread has its old scales by now)
#pragma unroll
        for (int w = 0; w < C8_WARPS; w++) { mk = fmaxf(mk, red_k[w]); mv = fmaxf(mv, red_v[w]); }
        const float sk = fmaxf(scale8_for<I8>(mk), was_k), sv = fmaxf(scale8_for<I8>(mv), was_v), ik = 1.0f / sk, iv = 1.0f / sv;
        const int dk = a.dim_ld, dv = a.vdim_ld;
        uint8_t* kd = static_cast<uint8_t*>(a.k_pool) + (((size_t)page * a.block_size + in_page - off) * a.kv_heads + h) * dk;
        uint8_t* vd = static_cast<uint8_t*>(a.v_pool) + (((size_t)page * a.block_size + in_page - off) * a.kv_heads + h) * dv;
#pragma unroll
        for (int i = 0; i < C8_ROWS; i++) {
            const int j = warp + i * C8_WARPS;
            if (j >= n) continue;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int d = 4 * lane + 128 * e;
                if (d < dk) *reinterpret_cast<uint32_t*>(kd + (size_t)(off + j) * a.kv_heads * dk + d) = pack8<I8>(k[i][e].x * ik, k[i][e].y * ik, k[i][e].z * ik, k[i][e].w * ik);
                if (d < dv) *reinterpret_cast<uint32_t*>(vd + (size_t)(off + j) * a.kv_heads * dv + d) = pack8<I8>(v[i][e].x * iv, v[i][e].y * iv, v[i][e].z * iv, v[i][e].w * iv);
            }
        }
        if (off && (sk != was_k || sv != was_v)) {
            const int kc = dk >> 4, vc = dv >> 4;
            for (int i = threadIdx.x; i < off * (kc + vc); i += C8_THREADS) {
                const int t = i / (kc + vc), c = i - t * (kc + vc);
                const bool key = c < kc;
                const float ratio = key ? was_k / sk : was_v / sv;
                if (ratio == 1.0f) continue;
                uint4* dst = reinterpret_cast<uint4*>(key ? kd + (size_t)t * a.kv_heads * dk + c * 16 : vd + (size_t)t * a.kv_heads * dv + (c - kc) * 16);
                uint4 u = *dst;
                u.x = rescale8<I8>(u.x, ratio); u.y = rescale8<I8>(u.y, ratio); u.z = rescale8<I8>(u.z, ratio); u.w = rescale8<I8>(u.w, ratio);
                *dst = u;
            }
        }
        if (threadIdx.x == 0) { a.k_scale[group] = sk; a.v_scale[group] = sv; }
        r += n;
    }
}

}  // namespace

int cmlb_cache8_append(const cmlb200_attn* a, float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int first, int rows, bool rotate, bool queries,
                       cudaStream_t st) {
    const bool q = queries && (a->q_norm || (rotate && a->freq) || (!rotate && a->temp_every > 0.f));
    const int span = rows > 256 ? kScaleTokens : 1;    // a CTA a row while that makes few; then one for the rows that make a whole group
    const dim3 grid((rows + span - 1) / span, a->kv_heads + (q ? 1 : 0));
    CMLB_REQUIRE(grid.y <= 65535, "8-bit cache: %d key/value heads", a->kv_heads);
    const bool vec = a->dim % 4 == 0 && a->vdim % 4 == 0 && ld % 4 == 0 && ((uintptr_t)d_qkv & 15) == 0, wide = a->dim_ld > 128 || a->vdim_ld > 128;
#define C8_LAUNCH(I8, N, V) CMLB_CUDA(launch_chain(cache8_append_kernel<I8, N, V>, grid, dim3(C8_THREADS), 0, 1, st, *a, d_qkv, ld, d_row_pos, d_row_slot, first, rows, span, (int)rotate))
#define C8_SIZE(I8, V) do { if (wide) C8_LAUNCH(I8, 2, V); else C8_LAUNCH(I8, 1, V); } while (0)
#define C8_FORM(I8) do { if (vec) C8_SIZE(I8, true); else C8_SIZE(I8, false); } while (0)
    if (a->cache_dtype == CMLB200_DT_I8) C8_FORM(true);
    else C8_FORM(false);
#undef C8_FORM
#undef C8_SIZE
#undef C8_LAUNCH
    return CMLB200_OK;
}
