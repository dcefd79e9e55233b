// Prompt portions over 8-bit caches where there are tiles enough for all SMs: as attention8_tiles.cu, but a CTA takes four query heads of a key/value head, two
// blocks of 128 rows that share the expansion of the codes. A key tile of a block costs the tensor cores 1,024 cycles and its exponentials as many of the
// special function units, so the two have to overlap: while one block's softmax runs, the other's products do.
//   0 .. 7    softmax, a thread a row, warps 0 .. 3 the first block's; a thread holds its 128 scores and hands the weights over in two halves
//   8 .. 11   expansion of a tile's keys, then of its values (the next tile's keys are requested ahead of this one's values, and the other way round)
//   12        issues tcgen05.mma, block by block: P V of a tile, then the scores of the next over them. Products are done in order, so that a block's scores being
//             there means that its O is at rest too
// Tensor memory: 128 columns of scores a block, then the blocks' O.
#include "attention8_tiles.cuh"

namespace {

// S: slabs of 64 dimensions of keys and values. Registers: 128 a thread at launch, then 176 x 256 + 104 x 128 + 56 x 128 = 128 x 512.
template <int S>
struct W8 {
    static constexpr int kSoft = 8, kConv = 4, kThreads = 32 * (kSoft + kConv + 4), kRows = 2 * T8_ROWS;
    static constexpr int kQ = 2 * S * T8_ROWS * 128, kK = S * T8_SLAB, kV = S * T8_SLAB, kStages = 2;
    static constexpr int kSmall = 1024 + 4 * kRows, kBytes = 1024 + kQ + kStages * (kK + kV) + kSmall;
};
constexpr int W8_TMEM = 512, W8_O_COL = 256, W8_SOFT_REGS = 176, W8_CONV_REGS = 104, W8_ISSUE_REGS = 56;

// grid = (kv_heads * blocks, tiles); a block is four query heads.
template <bool I8, int S, bool SLOPES>
__global__ void __launch_bounds__(W8<S>::kThreads, 1)
attention8_wide_kernel(const cmlb200_attn a, const float* __restrict__ qkv, int ld, const int4* __restrict__ tiles, __nv_bfloat16* __restrict__ out, int out_ld, int* status) {
    using C = W8<S>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const int dk = a.dim_ld, dv = a.vdim_ld;
    uint8_t* small = smem + C::kQ + C::kStages * (C::kK + C::kV);
    const uint32_t qs = smem_addr(smem), ks = qs + C::kQ, vs = ks + C::kStages * C::kK, bars = smem_addr(small);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto s_full = [&](int m) { return bars + 64 + 8 * m; };
    auto p_full = [&](int m, int half) { return bars + 80 + 16 * m + 8 * half; };
    const uint32_t drained = bars + 112;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(small + 128);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(small + 136);
    float* scales = reinterpret_cast<float*>(small + 256);                    // [4][2][T8_GROUPS]: key scales, log2 of value scales (tile i in i & 3)
    float* unit_s = reinterpret_cast<float*>(small + 1024);                   // [256] powers of two of the queries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConv = C::kSoft, kIssue = C::kSoft + C::kConv;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full(s), C::kConv); mbar_init(k_empty(s), 1); mbar_init(v_full(s), C::kConv); mbar_init(v_empty(s), 1);
            mbar_init(s_full(s), 1); mbar_init(p_full(s, 0), 4); mbar_init(p_full(s, 1), 4);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((uint32_t)W8_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dep_wait();
    const int4 tl = tiles[gridDim.y - 1 - blockIdx.y];                       // a prompt's last tiles, which see most keys, come first
    const int group = a.heads / a.kv_heads, blocks = gridDim.x / a.kv_heads, kh = blockIdx.x / blocks, hb = blockIdx.x % blocks * 4;
    const int n = tl.y, p0 = tl.w, p_last = p0 + n - 1, shift = __ffs(a.block_size) - 1;
    const int* table = a.block_table + (size_t)tl.z * a.table_ld;
    const T8Keys keys(a, p0, p_last, 0, 1);
    const int count = keys.count;
    t8_queries<S, C::kRows, C::kThreads / 32>(a, qkv, ld, tl, n, kh, hb, group, smem, unit_s);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    dep_trigger();                                     // a launch that allocates tensor memory too may start from here on: every CTA of this one has its own

    if (warp < kConv) {                                // ---- softmax
        more_registers<W8_SOFT_REGS>();
        const int m = warp >> 2, r = (warp & 3) * 32 + lane, i_tok = r & 63, h = hb + 2 * m + (r >> 6);
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_at = lanes + m * T8_KEYS, o_at = lanes + W8_O_COL + m * (S * 64);
        const bool live = i_tok < n && h < group;
        // (rows that are none have queries of zero and see what the last one sees; nobody looks at theirs)
        const int p = live ? p0 + i_tok : p_last, lo = first_key8(a, p), lo_last = first_key8(a, p_last), head = kh * group + (live ? h : 0);
        const float unit = unit_s[m * T8_ROWS + r], slope = SLOPES && live ? a.slopes[head] * kLog2e : 0.f;
        float ref = -INFINITY, l = 0.f, vref = -INFINITY;
        bool ok = true;
        for (int i = 0; i < count; i++) {
            const int kt = keys.start(i);
            ok = __all_sync(0xffffffffu, mbar_wait(s_full(m), i & 1, abort_flag, 1, status));
            if (!ok) break;
            tmem_fence_after();
            uint32_t v[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32_begin(s_at + 32 * c, v[c]);
            const float* sc = scales + (i & 3) * 2 * T8_GROUPS;
            float vm = vref, mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < T8_GROUPS; g++) vm = fmaxf(vm, sc[T8_GROUPS + g]);
            const float far = SLOPES ? slope * (float)(kt - p) : 0.f;        // the part of the bias that all keys share
            // (a scale times a query's power of two that underflows would make NaN of a masked score)
            auto factor = [&](int g) { return fmaxf(unit * sc[g], 1.17549435e-38f); };
            tmem_ld_wait(v);
            // unless every row of the CTA sees every key of the tile
            if (kt + T8_KEYS - 1 > p0 || (kt < lo_last && kt + T8_KEYS > a.keep)) {
                const int last = p - kt, begin = lo - kt, kept = a.keep - kt;
#pragma unroll
                for (int j = 0; j < T8_KEYS; j++) {
                    const bool hidden = (j > last) | ((j < begin) & (j >= kept));
                    v[j >> 5][j & 31] = hidden ? 0xff800000u : v[j >> 5][j & 31];
                }
            }
#pragma unroll
            for (int g = 0; g < T8_GROUPS; g++) mx = fmaxf(mx, t8_group_max<SLOPES>(v[g >> 1], g & 1, factor(g), slope, 16 * g));
            mx += far;
            if (__any_sync(0xffffffffu, mx > ref + kLazy || vm > vref)) {
                const float nm = fmaxf(ref, mx), c = nm == -INFINITY ? 1.f : ex2(ref - nm), cv = ex2(vref - vm);
                ref = nm;
                vref = vm;
                l *= c;
                if (i > 0) t8_scale_o(o_at, 0, 16, dv, c * cv);
            }
            const float u = (ref == -INFINITY ? 0.f : ref) - far;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int g = 2 * c + e;
                    const float bits = fmaxf(sc[T8_GROUPS + g] - vref, kFarScale) + kWeightBits;
                    l = fmaf(t8_group_weights<SLOPES>(v[c], w, e, factor(g), bits - u, slope, 16 * g), ex2(-bits), l);
                }
                tmem_st16(s_at + 16 * c, w);           // over the scores, which are all in registers
                if (c & 1) {                           // half of the tile's keys: their product may begin
                    tmem_st_wait();
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(m, c >> 1));
                }
            }
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(drained, 0, abort_flag, 2, status));
        tmem_fence_after();
        const float* row = qkv + (size_t)(tl.x + (live ? i_tok : 0)) * ld;
        if (a.sink && l > 0.f) l += ex2((a.sinks ? a.sinks[head] : 0.f) * kLog2e - ref);
        float inv = ok && l > 0.f ? ex2(vref - kWeightBits) * (a.out_scale == 0.f ? 1.f : a.out_scale) / l : 0.f;
        if (a.gate_col >= 0 && !a.gate_wide && live) inv *= sigmoidf(row[a.gate_col + head]);
        t8_write_row(a, o_at, 0, 32, live, inv, row, head, out, out_ld, (size_t)tl.x + (live ? i_tok : 0));
        tmem_fence_before();
    } else if (warp < kIssue) {                        // ---- expansion
        fewer_registers<W8_CONV_REGS>();
        const int tid = threadIdx.x - kConv * 32;
        T8Team<I8, S> k, v;
        k.init(a.k_pool, kh, a.kv_heads, dk, ks, tid);
        v.init(a.v_pool, kh, a.kv_heads, dv, vs, tid);
        // its first warp looks after the scales: lanes 0 .. 7 a group's key scale, 8 .. 15 its value scale
        const bool scaler = warp == kConv && lane < 2 * T8_GROUPS;
        auto scale_at = [&](int token) { return scaler ? (lane < T8_GROUPS ? a.k_scale : a.v_scale)[(size_t)token / kScaleTokens * a.kv_heads + kh] : 0.f; };
        bool ok = true;
        int next = 0, tok[4];
        const int at = t8_place(a, table, shift, keys, 0, lane);
        float scale = scale_at(at);
        t8_tokens(tok, at, keys.start(0), p_last, k.g0, k.in_group);
        k.load(tok, 0);
        v.load(tok, 0);
        if (count > 1) next = t8_place(a, table, shift, keys, 1, lane);
        for (int i = 0; i < count; i++) {
            const int st = i & 1, par = ((i >> 1) & 1) ^ 1;
            ok = __all_sync(0xffffffffu, mbar_wait(k_empty(st), par, abort_flag, 4, status));
            if (!ok) break;
            // (the scores of tile i - 2, which are done, were issued once the softmax of tile i - 3 was)
            if (scaler) scales[(i & 3) * 2 * T8_GROUPS + lane] = lane < T8_GROUPS ? scale : log2f(fmaxf(scale, 1.17549435e-38f));
            k.store_tile(tok, st * C::kK);
            if (lane == 0) mbar_arrive(k_full(st));
            if (i + 1 < count) {
                scale = scale_at(next);
                t8_tokens(tok, next, keys.start(i + 1), p_last, k.g0, k.in_group);
                k.load(tok, 0);
                if (i + 2 < count) next = t8_place(a, table, shift, keys, i + 2, lane);
            }
            ok = __all_sync(0xffffffffu, mbar_wait(v_empty(st), par, abort_flag, 5, status));
            if (!ok) break;
            v.store_tile(tok, st * C::kV);             // (one batch: `tok` is the next tile's by now)
            if (lane == 0) mbar_arrive(v_full(st));
            if (i + 1 < count) v.load(tok, 0);
        }
        __syncwarp();
    } else {                                           // ---- products
        fewer_registers<W8_ISSUE_REGS>();
        if (warp == kIssue) {
            // fp16 operands, fp32 accumulators, 128 rows; the second one takes V with its columns contiguous
            const uint32_t is = (1u << 4) | ((uint32_t)(T8_KEYS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t io = (1u << 4) | (1u << 16) | ((uint32_t)(dv >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int steps = dk >> 4;
            bool ok = true;
            auto keys_there = [&](int i) {
                ok = __all_sync(0xffffffffu, mbar_wait(k_full(i & 1), (i >> 1) & 1, abort_flag, 6, status));
                tmem_fence_after();
            };
            auto scores = [&](int m, int i) {
                if (elect_one()) {
                    const uint64_t ad = make_desc(qs + m * (S * T8_ROWS * 128)), bd = make_desc(ks + (i & 1) * C::kK);
                    const uint32_t alo = (uint32_t)ad, blo = (uint32_t)bd, hi = (uint32_t)(ad >> 32);
#pragma unroll
                    for (int k = 0; k < 4 * S; k++)
                        if (k < steps) umma_lo(tm + m * T8_KEYS, alo + (k >> 2) * (T8_ROWS * 128 >> 4) + 2 * (k & 3), blo + (k >> 2) * (T8_SLAB >> 4) + 2 * (k & 3), hi, is, k ? 1u : 0u);
                    if (m == 1) umma_commit(k_empty(i & 1));
                    umma_commit(s_full(m));
                }
                __syncwarp();
            };
            keys_there(0);
            for (int m = 0; m < 2 && ok; m++) scores(m, 0);
            for (int i = 0; i < count && ok; i++) {
                ok = __all_sync(0xffffffffu, mbar_wait(v_full(i & 1), (i >> 1) & 1, abort_flag, 7, status));
                for (int m = 0; m < 2 && ok; m++) {
                    const uint64_t vd = make_desc_mn(vs + (i & 1) * C::kV, T8_SLAB);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(p_full(m, half), i & 1, abort_flag, 8, status));
                        if (!ok) break;
                        tmem_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; k++)
                                umma_ts(tm + W8_O_COL + m * (S * 64), tm + m * T8_KEYS + 8 * k, (uint32_t)vd + k * (2048 >> 4), (uint32_t)(vd >> 32), io, (i | k) ? 1u : 0u);
                            if (half && m == 1) umma_commit(v_empty(i & 1));
                        }
                        __syncwarp();
                    }
                    if (ok && i + 1 < count) {
                        if (m == 0) keys_there(i + 1);
                        if (ok) scores(m, i + 1);
                    }
                }
            }
            // nothing that was issued outlives the CTA's tensor memory
            if (elect_one()) umma_commit(drained);
            __syncwarp();
            for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(drained, 0); it++) {}
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp == kIssue) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)W8_TMEM) : "memory");
    }
}

template <bool I8, int S, bool SLOPES>
int launch_wide(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, int* status, cudaStream_t st) {
    using C = W8<S>;
    const int blocks = (a->heads / a->kv_heads + 3) / 4;
    CMLB_REQUIRE((long long)a->kv_heads * blocks < (1LL << 31) && tiles <= 65535, "cmlb200_attention_tiles: %d tiles, %d heads", tiles, a->heads);
    static size_t attr[kMaxDevices] = {};
    auto kern = attention8_wide_kernel<I8, S, SLOPES>;
    const size_t smem = C::kBytes > 118 * 1024 ? C::kBytes : 118 * 1024;     // one CTA to an SM: each needs all of its tensor memory
    CMLB_CUDA(cmlb_ensure_smem(kern, smem, attr));
    CMLB_CUDA(launch_chain(kern, dim3(a->kv_heads * blocks, tiles), dim3(C::kThreads), smem, 1, st, *a, d_qkv, ld, (const int4*)d_tiles, d_out, out_ld, status));
    return CMLB200_OK;
}

}  // namespace

// A key/value head has to have more than two query heads, and there have to be CTAs for all SMs.
bool cmlb_attention8_wide_fits(const cmlb200_attn* a, int tiles) {
    const int group = a->heads / a->kv_heads;
    return a->dim_ld <= 128 && a->vdim_ld <= 128 && group > 2 && (long long)tiles * a->kv_heads * ((group + 3) / 4) >= cmlb_num_sms();
}

int cmlb_attention8_wide(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, int* status, cudaStream_t st) {
    const int widest = a->dim_ld > a->vdim_ld ? a->dim_ld : a->vdim_ld;
#define W8_ARGS a, d_qkv, ld, d_tiles, tiles, d_out, out_ld, status, st
#define W8_FORM(I8, S) return a->slopes ? launch_wide<I8, S, true>(W8_ARGS) : launch_wide<I8, S, false>(W8_ARGS)
#define W8_SIZES(I8)                        \
    do {                                    \
        if (widest <= 64) W8_FORM(I8, 1);   \
        W8_FORM(I8, 2);                     \
    } while (0)
    if (a->cache_dtype == CMLB200_DT_I8) W8_SIZES(true);
    W8_SIZES(false);
#undef W8_SIZES
#undef W8_FORM
#undef W8_ARGS
}
