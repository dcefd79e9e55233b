// Prompt portions over 8-bit caches where there are tiles enough for all SMs: as attention8_tiles.cu, but a CTA takes four query heads of a key/value head, two
// blocks of 128 rows that share the expansion of the codes. A key tile of a block costs the tensor cores 1,024 cycles and its exponentials as many of the
// special function units, so products and softmax have to overlap: a block has two accumulators of scores, 64 keys each, and while the weights of one half tile
// are made, the scores of the next and the other block's products are.
//   0 .. 7    softmax, a thread a row, warps 0 .. 3 the first block's
//   8 .. 15   expansion, four warps for keys and four for values (the next tile's codes are requested once this one's are written)
//   16, 17    issue tcgen05.mma, a block each: the scores of half tile j + 1, then P V of half tile j
// Measured with 8 heads of 128 and 4 queries each: 4,096 rows behind 4,096 tokens 494 us, 835 TFLOP/s (489 as e4m3); 2,048 rows without a cache 55.6 us. Bound by the chain of a softmax
// warp, and by score products of 64 keys: 6 KB of operands from shared memory are 48 cycles of its 128 bytes, the product itself 32. (Counters: the tensor
// cores' own pipe active half of the time, products 38 %.) 80 registers a thread of the expansion are a third of what is shared out; with fewer warps there, softmax threads could hold 128 keys.
// Where a key/value head has 5 or 6 query heads, the second CTA's second block has none and is computed all the same (2,048 rows, 8 key/value heads: 113 us and 115).
// Tensor memory: a block's 2 x 64 columns of scores, over which its weights lie, then the blocks' O.
#include "attention8_tiles.cuh"

namespace {

// S: slabs of 64 dimensions of keys and values. Registers: 96 a thread at launch, then 128 x 256 + 80 x 256 + 64 x 128 = 96 x 640.
template <int S>
struct W8 {
    static constexpr int kSoft = 8, kConv = 4, kThreads = 32 * (kSoft + 2 * kConv + 4), kRows = 2 * T8_ROWS;
    static constexpr int kQ = 2 * S * T8_ROWS * 128, kK = S * T8_SLAB, kV = S * T8_SLAB, kStages = 2;
    static constexpr int kSmall = 1024 + 4 * kRows, kBytes = 1024 + kQ + kStages * (kK + kV) + kSmall;
};
constexpr int W8_TMEM = 512, W8_O_COL = 256, W8_SOFT_REGS = 128, W8_CONV_REGS = 80, W8_ISSUE_REGS = 64;

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
    auto s_full = [&](int m, int half) { return bars + 64 + 16 * m + 8 * half; };
    auto p_full = [&](int m, int half) { return bars + 96 + 16 * m + 8 * half; };
    auto pv_done = [&](int m) { return bars + 128 + 8 * m; };
    auto drained = [&](int m) { return bars + 144 + 8 * m; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(small + 192);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(small + 200);
    float* scales = reinterpret_cast<float*>(small + 256);                    // [4][T8_SCALES] (tile i in i & 3)
    float* unit_s = reinterpret_cast<float*>(small + 1024);                   // [256] powers of two of the queries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConv = C::kSoft, kIssue = C::kSoft + 2 * C::kConv;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full(s), C::kConv); mbar_init(k_empty(s), 2); mbar_init(v_full(s), C::kConv); mbar_init(v_empty(s), 2);
            mbar_init(s_full(s, 0), 1); mbar_init(s_full(s, 1), 1); mbar_init(p_full(s, 0), 4); mbar_init(p_full(s, 1), 4); mbar_init(pv_done(s), 1); mbar_init(drained(s), 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((uint32_t)W8_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dep_wait();
    const int4 tl = tiles[gridDim.y - 1 - blockIdx.y];                       // a prompt's last tiles, which see most keys, come first
    const int group = a.heads / a.kv_heads, blocks = gridDim.x / a.kv_heads, kh = blockIdx.x / blocks;
    const int n = tl.y, p0 = tl.w, p_last = p0 + n - 1, shift = __ffs(a.block_size) - 1;
    if (n <= 0) {                                      // (as the form for few tiles does)
        __syncthreads();
        if (warp == kIssue) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"((uint32_t)W8_TMEM) : "memory");
        return;
    }
    const T8Heads rows = {n, group, (int)(blockIdx.x % blocks) * 4};
    const int* table = a.block_table + (size_t)tl.z * a.table_ld;
    const T8Keys keys(a, p0, p_last, 0, 1);
    // half tiles; the last one is left out where it lies behind the last row
    const int count = keys.count, halves = 2 * count - (keys.start(count - 1) + 64 > p_last ? 1 : 0);
    t8_queries<S, C::kRows, C::kThreads / 32>(a, qkv, ld, tl, rows, kh, smem, unit_s, warp);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    dep_trigger();                                     // a launch that allocates tensor memory too may start from here on: every CTA of this one has its own

    if (warp < kConv) {                                // ---- softmax
        more_registers<W8_SOFT_REGS>();
        const int m = warp >> 2, r = (warp & 3) * 32 + lane;
        int i_tok, h;
        const bool live = rows.find(m * T8_ROWS + r, i_tok, h);
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), o_at = lanes + W8_O_COL + m * (S * 64);
        // (rows that are none have queries of zero and see what the last one sees; nobody looks at theirs)
        const int p = live ? p0 + i_tok : p_last, lo = first_key8(a, p), lo_last = first_key8(a, p_last), head = kh * group + (live ? h : 0);
        const float unit = unit_s[m * T8_ROWS + r], slope = SLOPES && live ? a.slopes[head] * kLog2e : 0.f;
        float ref = -INFINITY, wref = -INFINITY, l = 0.f;                    // references: log2 of scores, log2 of scores times value scales
        bool ok = true;
        for (int j = 0; j < halves; j++) {
            const int half = j & 1, kt = keys.start(j >> 1) + 64 * half;    // the first key
            const uint32_t s_at = lanes + m * T8_KEYS + 64 * half;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full(m, half), (j >> 1) & 1, abort_flag, 1, status));
            if (!ok) break;
            tmem_fence_after();
            uint32_t v[2][32];
            tmem_ld32_begin(s_at, v[0]);
            tmem_ld32_begin(s_at + 32, v[1]);
            const float* sc = scales + ((j >> 1) & 3) * T8_SCALES + 4 * half;
            const float4 s4 = *reinterpret_cast<const float4*>(sc), l4 = *reinterpret_cast<const float4*>(sc + T8_GROUPS);
            // (a scale times a query's power of two that underflows would make NaN of a masked score)
            const float f[4] = {fmaxf(unit * s4.x, 1.17549435e-38f), fmaxf(unit * s4.y, 1.17549435e-38f), fmaxf(unit * s4.z, 1.17549435e-38f), fmaxf(unit * s4.w, 1.17549435e-38f)};
            const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
            const float far = SLOPES ? slope * (float)(kt - p) : 0.f;        // the part of the bias that all keys share
            tmem_ld_wait(v);
            // unless every row of the CTA sees every one of these keys
            if (kt + 63 > p0 || (kt < lo_last && kt + 64 > a.keep)) {
                const int last = p - kt, begin = lo - kt, kept = a.keep - kt;
#pragma unroll
                for (int k = 0; k < 64; k++) {
                    const bool hidden = (k > last) | ((k < begin) & (k >= kept));
                    v[k >> 5][k & 31] = hidden ? 0xff800000u : v[k >> 5][k & 31];
                }
            }
            float mx = -INFINITY, mw = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float most = t8_group_max<SLOPES>(v[g >> 1], g & 1, f[g], slope, 16 * g);
                mx = fmaxf(mx, most);
                mw = fmaxf(mw, most + lv[g]);
            }
            mx += far;
            mw += far;
            if (__any_sync(0xffffffffu, mx > ref + kLazy || mw > wref + kLazy)) {
                const float nm = fmaxf(ref, mx), nw = fmaxf(wref, mw), c = nw == -INFINITY ? 1.f : ex2(wref - nw);
                l *= nm == -INFINITY ? 1.f : ex2(ref - nm);
                ref = nm;
                wref = nw;
                if (j > 0) {
                    // (these scores were issued behind P V of half tile j - 2, so that one is done)
                    ok = __all_sync(0xffffffffu, mbar_wait(pv_done(m), (j - 1) & 1, abort_flag, 3, status));
                    if (!ok) break;
                    tmem_fence_after();
                    t8_scale_o(o_at, 0, 16, dv, c);
                }
            }
            const float lift = ref == -INFINITY ? 0.f : wref - ref, u = (ref == -INFINITY ? 0.f : ref) - far;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int g = 2 * c + e;
                    const float bits = fmaxf(lv[g] - lift, kFarScale) + kWeightBits;
                    l = fmaf(t8_group_weights<SLOPES>(v[c], w, e, f[g], bits - u, slope, 16 * g), ex2(-bits), l);
                }
                tmem_st16(s_at + 16 * c, w);           // over the scores, which are all in registers
            }
            tmem_st_wait();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(m, half));
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(drained(m), 0, abort_flag, 2, status));
        tmem_fence_after();
        const float* row = qkv + (size_t)(tl.x + (live ? i_tok : 0)) * ld;
        if (a.sink && l > 0.f) l += ex2((a.sinks ? a.sinks[head] : 0.f) * kLog2e - ref);
        float inv = ok && l > 0.f ? ex2(wref - ref - kWeightBits) * (a.out_scale == 0.f ? 1.f : a.out_scale) / l : 0.f;
        if (a.gate_col >= 0 && !a.gate_wide && live) inv *= sigmoidf(row[a.gate_col + head]);
        t8_write_row(a, o_at, 0, 32, live, inv, row, head, out, out_ld, (size_t)tl.x + (live ? i_tok : 0));
        tmem_fence_before();
    } else if (warp < kIssue) {                        // ---- expansion
        fewer_registers<W8_CONV_REGS>();
        const bool key = warp < kConv + C::kConv;
        T8Team<I8, S, S == 1 ? 4 : 8> team;
        team.init(key ? a.k_pool : a.v_pool, kh, a.kv_heads, key ? dk : dv, key ? ks : vs, threadIdx.x - (key ? kConv : kConv + C::kConv) * 32);
        const int stage_bytes = key ? C::kK : C::kV;
        T8Scaler scaler = {warp == kConv && lane < 2 * T8_GROUPS, lane, kh, 0.f};
        bool ok = true;
        int next = 0, tok[4];
        const int at = t8_place(a, table, shift, keys, 0, lane);
        scaler.fetch(a, at);
        t8_tokens(tok, at, keys.start(0), p_last, team.g0, team.in_group);
        team.load(tok, 0);
        if (count > 1) next = t8_place(a, table, shift, keys, 1, lane);
        for (int i = 0; i < count; i++) {
            const int st = i & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(key ? k_empty(st) : v_empty(st), ((i >> 1) & 1) ^ 1, abort_flag, key ? 4 : 5, status));
            if (!ok) break;
            // (the scores of tile i - 2, which are done, were issued once the softmax of tile i - 4 was)
            scaler.put(scales, i);
            team.store_tile(tok, st * stage_bytes);
            if (lane == 0) mbar_arrive(key ? k_full(st) : v_full(st));
            if (i + 1 < count) {
                scaler.fetch(a, next);
                t8_tokens(tok, next, keys.start(i + 1), p_last, team.g0, team.in_group);
                team.load(tok, 0);
                if (i + 2 < count) next = t8_place(a, table, shift, keys, i + 2, lane);
            }
        }
        __syncwarp();
    } else {                                           // ---- products
        fewer_registers<W8_ISSUE_REGS>();
        if (warp < kIssue + 2) {
            // fp16 operands, fp32 accumulators, 128 rows; the second one takes V with its columns contiguous
            const uint32_t is = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t io = (1u << 4) | (1u << 16) | ((uint32_t)(dv >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const int m = __shfl_sync(0xffffffffu, warp - kIssue, 0), steps = dk >> 4;
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), s_at = tm + m * T8_KEYS, o_at = tm + W8_O_COL + m * (S * 64);
            bool ok = true;
            auto scores = [&](int j) {
                const int st = (j >> 1) & 1, half = j & 1;
                if (!half) ok = __all_sync(0xffffffffu, mbar_wait(k_full(st), (j >> 2) & 1, abort_flag, 6, status));
                if (!ok) return;
                tmem_fence_after();
                if (elect_one()) {
                    const uint64_t ad = make_desc(qs + m * (S * T8_ROWS * 128)), bd = make_desc(ks + st * C::kK + half * (64 * 128));
                    const uint32_t alo = (uint32_t)ad, blo = (uint32_t)bd, hi = (uint32_t)(ad >> 32), d = s_at + 64 * half;
#pragma unroll
                    for (int k = 0; k < 4 * S; k++)
                        if (k < steps) umma_lo(d, alo + (k >> 2) * (T8_ROWS * 128 >> 4) + 2 * (k & 3), blo + (k >> 2) * (T8_SLAB >> 4) + 2 * (k & 3), hi, is, k ? 1u : 0u);
                    if (half) umma_commit(k_empty(st));
                    umma_commit(s_full(m, half));
                }
                __syncwarp();
            };
            scores(0);
            for (int j = 0; j < halves && ok; j++) {
                const int st = (j >> 1) & 1, half = j & 1;
                if (j + 1 < halves) scores(j + 1);     // into the accumulator whose weights' product has been issued
                if (ok && !half) ok = __all_sync(0xffffffffu, mbar_wait(v_full(st), (j >> 2) & 1, abort_flag, 7, status));
                ok = ok && __all_sync(0xffffffffu, mbar_wait(p_full(m, half), (j >> 1) & 1, abort_flag, 8, status));
                if (!ok) break;
                tmem_fence_after();
                if (elect_one()) {
                    const uint64_t vd = make_desc_mn(vs + st * C::kV + half * (64 * 128), T8_SLAB);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma_ts(o_at, s_at + 64 * half + 8 * k, (uint32_t)vd + k * (2048 >> 4), (uint32_t)(vd >> 32), io, (j | k) ? 1u : 0u);
                    if (half) umma_commit(v_empty(st));
                    umma_commit(pv_done(m));
                }
                __syncwarp();
            }
            // nothing that was issued outlives the CTA's tensor memory
            if (elect_one()) umma_commit(drained(m));
            __syncwarp();
            for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(drained(m), 0); it++) {}
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
