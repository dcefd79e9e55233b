// Prompt portions over 8-bit caches (cache8.cuh) on the 5th-generation tensor cores.
//
// A CTA takes a tile of up to 64 consecutive rows of one sequence and some of a key/value head's query heads, 128 rows of the products, and walks key
// tiles of 128 tokens: S = Q K^T into one of two accumulators in tensor memory, O += P V with P in tensor memory over the scores it came from. Roles, by warp:
//   0 .. 7    softmax, two threads a row with 64 keys each (the warps w and w + 4 meet for the row's largest score): all scores in registers, then
//             exponentials straight into P. The reference of the exponentials moves, and O is scaled, only when a row has grown by more than 8 (powers of two)
//   8 .. 15   expansion, four warps for keys and four for values: codes from the cache (the next tile's are requested once this one's are written) to fp16 in
//             shared memory, keys with the dimensions contiguous, values with theirs as the contiguous non-summed side, both with 128-byte swizzle. Codes are
//             exact in fp16; scales stay apart: a group's key scale multiplies its scores, its value scale joins the exponent of its weights
//   16        issues tcgen05.mma: the scores of tile i + 1, then P V of tile i, so that products and softmax overlap
// Rows are (head, token) pairs, one head after the other, so short tiles fill few blocks; queries are fp16 over a power of two of their own. A weight is 2^s times its group's value
// scale, over the largest such product that its row has met, times 128: at most 2^15, and never small because of values that the row does not see or passes over. That
// largest product and the largest score, which the sum of 2^(s - m) is relative to, are followed apart.
// Few tiles: a cluster of up to 8 CTAs splits the keys and merges through distributed shared memory.
// Keys behind a portion's last row are read as that row's (their weights are zero), so nothing other requests left can reach the sums. Every wait is
// bounded; one that gives up leaves a code in a status word in host memory, the products under way are waited for and tensor memory is freed.
// Few tiles are bound by latency: what comes before the first scores (table, codes, expansion, queries: 3 to 4 us), 1.2 (heads of 64) to 1.5 us a key tile of which
// 0.54 are exponentials, and the end. Heads of 128, 8 of 4 queries each: 64 rows 9.3 us, behind 6,000 tokens 24.5, 512 rows 14.2, 1,024 rows 28.3.
#include "attention8_tiles.cuh"
#include "status_word.cuh"

namespace {

// Stages of keys and of values, and the CTAs that share a tile's keys.
struct T8Plan {
    int stages, splits;
};
// Shared memory: queries, key stages, value stages, then the small things. S: slabs of 64 dimensions.
template <int S>
struct T8 {
    static constexpr int kSoft = 8, kConv = 4, kThreads = 32 * (kSoft + 2 * kConv + 4);
    static constexpr int kQ = S * T8_ROWS * 128, kK = S * T8_SLAB, kV = S * T8_SLAB;
    static constexpr int kSmall = 1024 + 4 * T8_ROWS * (1 + 8 + 2 * T8_SPLITS);
    static int bytes(int stages) { return 1024 + kQ + stages * (kK + kV) + kSmall; }
};
constexpr int T8_TMEM = 512, T8_O_COL = 256;
// registers of a thread: 96 at launch, then shared out by role (128 x 256 + 80 x 256 + 64 x 128 = 96 x 640)
constexpr int T8_SOFT_REGS = 128, T8_CONV_REGS = 80, T8_ISSUE_REGS = 64;

// grid = (splits, kv_heads * blocks, tiles), clusters of `splits`; a block is 128 (head, token) rows; those behind a short tile's last end at once.
template <bool I8, int S, bool SLOPES>
__global__ void __launch_bounds__(T8<S>::kThreads, 1)
attention8_tiles_kernel(const cmlb200_attn a, const float* __restrict__ qkv, int ld, const int4* __restrict__ tiles, __nv_bfloat16* __restrict__ out, int out_ld, const T8Plan plan,
                        int* status) {
    using C = T8<S>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const int dk = a.dim_ld, dv = a.vdim_ld, stages = plan.stages, splits = plan.splits, rank = blockIdx.x;
    uint8_t* small = smem + C::kQ + stages * (C::kK + C::kV);
    const uint32_t qs = smem_addr(smem), ks = qs + C::kQ, vs = ks + stages * C::kK, bars = smem_addr(small);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto s_full = [&](int b) { return bars + 64 + 8 * b; };
    auto p_full = [&](int b) { return bars + 80 + 8 * b; };
    const uint32_t pv_done = bars + 96, drained = bars + 104;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(small + 128);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(small + 136);
    float* scales = reinterpret_cast<float*>(small + 256);                    // [4][T8_SCALES] (tile i in i & 3)
    float* unit_s = reinterpret_cast<float*>(small + 1024);                   // [128] powers of two of the queries
    float2* meet = reinterpret_cast<float2*>(unit_s + T8_ROWS);               // [2][2][128] the two halves' largest scores and products with value scales, at the end sums
    float* c_m = unit_s + 9 * T8_ROWS;                                         // [T8_SPLITS][128] maxima and sums of the whole cluster
    float* c_l = c_m + T8_SPLITS * T8_ROWS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConv = C::kSoft, kIssue = C::kSoft + 2 * C::kConv;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full(s), C::kConv); mbar_init(k_empty(s), 1); mbar_init(v_full(s), C::kConv); mbar_init(v_empty(s), 1);
            mbar_init(s_full(s), 1); mbar_init(p_full(s), C::kSoft);
        }
        mbar_init(pv_done, 1);
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((uint32_t)T8_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // first phase of the cluster's barrier: nothing is stored into another CTA before that one runs
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int group = a.heads / a.kv_heads, blocks = gridDim.y / a.kv_heads, kh = blockIdx.y / blocks, first_row = (int)(blockIdx.y % blocks) * T8_ROWS, shift = __ffs(a.block_size) - 1;
    dep_wait();
    dep_trigger();                                     // a launch that allocates tensor memory too may start from here on: every CTA of this one has its own
    const int4 tl = tiles[gridDim.z - 1 - blockIdx.z];                       // a prompt's last tiles, which see most keys, come first
    const int n = tl.y, p0 = tl.w, p_last = p0 + n - 1;
    const T8Rows rows(n, group, first_row);
    if (rows.none()) {                                 // (the whole cluster's; nothing has been issued)
        if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp == kIssue) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)T8_TMEM) : "memory");
        return;
    }
    const int* table = a.block_table + (size_t)tl.z * a.table_ld;
    const T8Keys keys(a, p0, p_last, rank, splits);
    const int count = keys.count;
    // the queries, by all warps but those of the expansion, which begin with the first keys meanwhile
    auto queries = [&](int w) {
        if (count > 0) t8_queries<S, T8_ROWS, C::kSoft + 4>(a, qkv, ld, tl, rows, kh, smem, unit_s, w);
        asm volatile("bar.sync 5, %0;" ::"n"(32 * (C::kSoft + 4)) : "memory");
    };

    if (warp < kConv) {                                // ---- softmax
        queries(warp);
        more_registers<T8_SOFT_REGS>();
        const int half = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        int i_tok, h;
        const bool live = rows.find(r, i_tok, h);
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), o_at = lanes + T8_O_COL;
        // (rows that are none have queries of zero and see what the last one sees; nobody looks at theirs)
        const int p = live ? p0 + i_tok : p_last, lo = first_key8(a, p), lo_last = first_key8(a, p_last), head = kh * group + (live ? h : 0);
        const float unit = unit_s[r], slope = SLOPES && live ? a.slopes[head] * kLog2e : 0.f;
        auto pair_meets = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };
        float ref = -INFINITY, wref = -INFINITY, l = 0.f;                    // references: log2 of scores, log2 of scores times value scales
        bool ok = true;
        for (int i = 0; i < count; i++) {
            const int kt = keys.start(i) + 64 * half, buf = i & 1;          // this thread's first key
            const uint32_t s_at = lanes + buf * T8_KEYS;
            ok = ok && __all_sync(0xffffffffu, mbar_wait(s_full(buf), (i >> 1) & 1, abort_flag, 1, status));
            uint32_t v[2][32];
            float mx = -INFINITY, mw = -INFINITY;
            const float* sc = scales + (i & 3) * T8_SCALES + 4 * half;
            const float far = SLOPES ? slope * (float)(kt - p) : 0.f;        // the part of the bias that all of its keys share
            float f[4], lv[4];                         // factors of its four groups' scores, log2 of their value scales
            if (ok) {
                tmem_fence_after();
#pragma unroll
                for (int c = 0; c < 2; c++) tmem_ld32_begin(s_at + 64 * half + 32 * c, v[c]);
                const float4 s4 = *reinterpret_cast<const float4*>(sc), l4 = *reinterpret_cast<const float4*>(sc + T8_GROUPS);
                // (a scale times a query's power of two that underflows would make NaN of a masked score)
                f[0] = fmaxf(unit * s4.x, 1.17549435e-38f); f[1] = fmaxf(unit * s4.y, 1.17549435e-38f); f[2] = fmaxf(unit * s4.z, 1.17549435e-38f); f[3] = fmaxf(unit * s4.w, 1.17549435e-38f);
                lv[0] = l4.x; lv[1] = l4.y; lv[2] = l4.z; lv[3] = l4.w;
                tmem_ld_wait(v);
                // unless every row of the CTA sees every one of these keys
                if (kt + 63 > p0 || (kt < lo_last && kt + 64 > a.keep)) {
                    const int last = p - kt, begin = lo - kt, kept = a.keep - kt;
#pragma unroll
                    for (int j = 0; j < 64; j++) {
                        const bool hidden = (j > last) | ((j < begin) & (j >= kept));
                        v[j >> 5][j & 31] = hidden ? 0xff800000u : v[j >> 5][j & 31];
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const float m = t8_group_max<SLOPES>(v[g >> 1], g & 1, f[g], slope, 16 * g);
                    mx = fmaxf(mx, m);
                    mw = fmaxf(mw, m + lv[g]);
                }
                mx += far;
                mw += far;
                meet[(2 * buf + half) * T8_ROWS + r] = make_float2(mx, mw);
            }
            tmem_fence_before();
            pair_meets();                              // both halves' scores are in registers, and their largest known
            tmem_fence_after();
            if (!ok) continue;                         // (the other half may have been luckier: the two meet once a tile whatever comes)
            const float2 other = meet[(2 * buf + (half ^ 1)) * T8_ROWS + r];
            mx = fmaxf(mx, other.x);
            mw = fmaxf(mw, other.y);
            if (__any_sync(0xffffffffu, mx > ref + kLazy || mw > wref + kLazy)) {
                const float nm = fmaxf(ref, mx), nw = fmaxf(wref, mw), c = nw == -INFINITY ? 1.f : ex2(wref - nw);
                l *= nm == -INFINITY ? 1.f : ex2(ref - nm);
                ref = nm;
                wref = nw;
                if (i > 0) {
                    // (scores of this tile were issued behind P V of tile i - 2, so that one is done)
                    ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (i - 1) & 1, abort_flag, 2, status));
                    if (!ok) continue;
                    tmem_fence_after();
                    t8_scale_o(o_at, 16 * half, 32, dv, c);
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
                tmem_st16(s_at + 32 * half + 16 * c, w);                      // over scores that both halves have in registers
            }
            tmem_st_wait();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(buf));
        }
        if (ok && count > 0) ok = __all_sync(0xffffffffu, mbar_wait(drained, 0, abort_flag, 3, status));
        tmem_fence_after();
        if (!ok) { ref = -INFINITY; l = 0.f; }
        const float lift = wref - ref;
        // a row's two sums (a tile's largest scores have been read before the next one's are written: two pairs of places)
        pair_meets();
        meet[half * T8_ROWS + r].x = l;
        pair_meets();
        l += meet[(half ^ 1) * T8_ROWS + r].x;
        const float* row = qkv + (size_t)(tl.x + (live ? i_tok : 0)) * ld;
        float mt = ref, sum = l;
        if (splits > 1) {
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            if (half == 0) {
#pragma unroll
                for (int s = 0; s < T8_SPLITS; s++)
                    if (s < splits) {
                        uint32_t am, al;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(am) : "r"(smem_addr(c_m + rank * T8_ROWS + r)), "r"(s));
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(al) : "r"(smem_addr(c_l + rank * T8_ROWS + r)), "r"(s));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(am), "f"(ref) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(al), "f"(l) : "memory");
                    }
            }
            __syncwarp();
            cluster_meet();
            sum = 0.f;
            for (int s = 0; s < splits; s++) mt = fmaxf(mt, c_m[s * T8_ROWS + r]);
            for (int s = 0; s < splits; s++) {
                const float ms = c_m[s * T8_ROWS + r];
                if (ms != -INFINITY) sum = fmaf(c_l[s * T8_ROWS + r], ex2(ms - mt), sum);
            }
        }
        if (a.sink && sum > 0.f) sum += ex2((a.sinks ? a.sinks[head] : 0.f) * kLog2e - mt);
        // what O is multiplied with: its unit, what this CTA's reference lacks of the row's, one over the sum, the gate
        float inv = ref != -INFINITY && sum > 0.f ? ex2(lift - kWeightBits) * ex2(ref - mt) * (a.out_scale == 0.f ? 1.f : a.out_scale) / sum : 0.f;
        if (a.gate_col >= 0 && !a.gate_wide && live) inv *= sigmoidf(row[a.gate_col + head]);
        if (splits == 1) {
            t8_write_row(a, o_at, 32 * half, 64, live, inv, row, head, out, out_ld, (size_t)tl.x + (live ? i_tok : 0));
            tmem_fence_before();
        } else {
            // this CTA's part of every row's result, over its operands (all of its products are done); then the cluster's CTAs add a share of the elements each
            float* Os = reinterpret_cast<float*>(smem) + (size_t)r * (dv + 4);
            const bool any = ref != -INFINITY;         // (a CTA that had no tile: its O may be anything)
#pragma unroll 1
            for (int c0 = 32 * half; c0 < dv; c0 += 64) {
                uint32_t o[32];
                if (count > 0) tmem_ld32(o_at + c0, o);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c0 + 4 * j < dv)
                        *reinterpret_cast<float4*>(Os + c0 + 4 * j) = any ? make_float4(__uint_as_float(o[4 * j]) * inv, __uint_as_float(o[4 * j + 1]) * inv, __uint_as_float(o[4 * j + 2]) * inv,
                                                                                        __uint_as_float(o[4 * j + 3]) * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            tmem_fence_before();
            __syncwarp();
            cluster_meet();
            const int quads = dv / 4;
            for (int e = rank * (32 * C::kSoft) + threadIdx.x; e < T8_ROWS * quads; e += splits * (32 * C::kSoft)) {
                const int k = e / quads, c = (e - k * quads) * 4;
                int tok, hh;
                if (!rows.find(k, tok, hh)) continue;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y[T8_SPLITS];
#pragma unroll
                for (int s = 0; s < T8_SPLITS; s++) {
                    y[s] = x;
                    if (s < splits) {
                        uint32_t ax;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ax) : "r"(smem_addr(reinterpret_cast<float*>(smem) + (size_t)k * (dv + 4) + c)), "r"(s));
                        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y[s].x), "=f"(y[s].y), "=f"(y[s].z), "=f"(y[s].w) : "r"(ax) : "memory");
                    }
                }
#pragma unroll
                for (int s = 0; s < T8_SPLITS; s++) { x.x += y[s].x; x.y += y[s].y; x.z += y[s].z; x.w += y[s].w; }
                const float z[4] = {x.x, x.y, x.z, x.w};
                const int hd = kh * group + hh;
                const float* gate = qkv + (size_t)(tl.x + tok) * ld + a.gate_col + hd * a.vdim + c;
                __nv_bfloat16* dst = out + (size_t)(tl.x + tok) * out_ld + (size_t)hd * a.vdim + c;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (c + j < a.vdim) dst[j] = __float2bfloat16_rn(a.gate_wide ? z[j] * sigmoidf(gate[j]) : z[j]);
            }
            __syncwarp();
            cluster_meet();                            // nobody leaves while others read its shared memory
        }
    } else {
        if (warp < kIssue) {                           // ---- expansion
            fewer_registers<T8_CONV_REGS>();
            const bool key = warp < kConv + C::kConv;
            T8Team<I8, S, S == 1 ? 4 : 8> team;
            team.init(key ? a.k_pool : a.v_pool, kh, a.kv_heads, key ? dk : dv, key ? ks : vs, threadIdx.x - (key ? kConv : kConv + C::kConv) * 32);
            const int stage_bytes = key ? C::kK : C::kV;
            bool ok = true;
            int st = 0, par = 1, next = 0, tok[4] = {0, 0, 0, 0};
            T8Scaler scaler = {warp == kConv && lane < 2 * T8_GROUPS, lane, kh, 0.f};
            if (count > 0) {
                const int at = t8_place(a, table, shift, keys, 0, lane);
                scaler.fetch(a, at);
                t8_tokens(tok, at, keys.start(0), p_last, team.g0, team.in_group);
                team.load(tok, 0);
                if (count > 1) next = t8_place(a, table, shift, keys, 1, lane);
            }
            for (int i = 0; i < count; i++) {
                ok = __all_sync(0xffffffffu, mbar_wait(key ? k_empty(st) : v_empty(st), par, abort_flag, key ? 4 : 5, status));
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
                if (++st == stages) { st = 0; par ^= 1; }
            }
        } else {                                       // ---- products
            queries(warp - 2 * C::kConv);
            fewer_registers<T8_ISSUE_REGS>();
            if (warp == kIssue && count > 0) {
                // fp16 operands, fp32 accumulators, 128 rows; the second one takes V with its columns contiguous
                const uint32_t is = (1u << 4) | ((uint32_t)(T8_KEYS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
                const uint32_t io = (1u << 4) | (1u << 16) | ((uint32_t)(dv >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
                const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
                const int steps = dk >> 4;
                int kst = 0, kpar = 0, vst = 0, vpar = 0;
                bool ok = true;
                auto scores = [&](int i) {
                    ok = __all_sync(0xffffffffu, mbar_wait(k_full(kst), kpar, abort_flag, 6, status));
                    if (!ok) return;
                    tmem_fence_after();
                    if (elect_one()) {
                        const uint64_t ad = make_desc(qs), bd = make_desc(ks + kst * C::kK);
                        const uint32_t alo = (uint32_t)ad, blo = (uint32_t)bd, hi = (uint32_t)(ad >> 32), d = tm + (i & 1) * T8_KEYS;
#pragma unroll
                        for (int k = 0; k < 4 * S; k++)
                            if (k < steps) umma_lo(d, alo + (k >> 2) * (T8_ROWS * 128 >> 4) + 2 * (k & 3), blo + (k >> 2) * (T8_SLAB >> 4) + 2 * (k & 3), hi, is, k ? 1u : 0u);
                        umma_commit(k_empty(kst));
                        umma_commit(s_full(i & 1));
                    }
                    __syncwarp();
                    if (++kst == stages) { kst = 0; kpar ^= 1; }
                };
                scores(0);
                for (int i = 0; i < count && ok; i++) {
                    if (i + 1 < count) scores(i + 1);      // into the other accumulator, whose weights' product has been issued
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(v_full(vst), vpar, abort_flag, 7, status));
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(p_full(i & 1), (i >> 1) & 1, abort_flag, 8, status));
                    if (!ok) break;
                    tmem_fence_after();
                    if (elect_one()) {
                        const uint64_t vd = make_desc_mn(vs + vst * C::kV, T8_SLAB);
                        const uint32_t p_at = tm + (i & 1) * T8_KEYS;
#pragma unroll
                        for (int k = 0; k < T8_KEYS / 16; k++)
                            umma_ts(tm + T8_O_COL, p_at + 8 * k, (uint32_t)vd + k * (2048 >> 4), (uint32_t)(vd >> 32), io, (i | k) ? 1u : 0u);
                        umma_commit(v_empty(vst));
                        umma_commit(pv_done);
                    }
                    __syncwarp();
                    if (++vst == stages) { vst = 0; vpar ^= 1; }
                }
                // nothing that was issued outlives the CTA's tensor memory
                if (elect_one()) umma_commit(drained);
                __syncwarp();
                for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(drained, 0); it++) {}
                __syncwarp();
            }
        }
        __syncwarp();
        if (splits > 1) {
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            cluster_meet();
            cluster_meet();
            cluster_meet();
        }
    }
    __syncthreads();
    if (warp == kIssue) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)T8_TMEM) : "memory");
    }
}

StatusWords<kMaxDevices> g_status8;

template <bool I8, int S, bool SLOPES>
int launch_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, int* status, cudaStream_t st) {
    using C = T8<S>;
    const int blocks = (a->heads / a->kv_heads + 1) / 2;
    CMLB_REQUIRE((long long)a->kv_heads * blocks <= 65535 && blocks < 32768 && tiles <= 65535, "cmlb200_attention_tiles: %d tiles, %d heads", tiles, a->heads);
    T8Plan plan;
    for (plan.stages = 2; plan.stages > 1 && C::bytes(plan.stages) > 227 * 1024; plan.stages--) {}
    // one CTA to an SM: each needs all of the SM's tensor memory, and a cluster's CTAs wait for one another
    const size_t need = (size_t)C::bytes(plan.stages), smem = need > 118 * 1024 ? need : 118 * 1024;
    static size_t attr[kMaxDevices] = {};
    static int room[kMaxDevices][T8_SPLITS + 1] = {};
    auto kern = attention8_tiles_kernel<I8, S, SLOPES>;
    CMLB_CUDA(cmlb_ensure_smem(kern, smem, attr));
    // How many CTAs share the keys of a tile: what takes least by an estimate in units of a key tile's time (1.7 us at heads of 128): 5 for a CTA's beginning and end
    // and 2 for a merge, times the waves, where clusters of a size share the device with as many as fit its groups of SMs. A block table's row bounds the keys.
    // (64 rows behind 6,000 tokens, 16 tiles of heads: clusters of 8 run in two waves, 43 us.)
    const long long ctas = (long long)tiles * a->kv_heads * blocks, reach = a->chunk > 0 ? a->chunk + 64 : a->window > 0 ? a->window + 64 : 0;
    long long keys = (long long)a->table_ld * a->block_size;
    if (reach && reach + a->keep < keys) keys = reach + a->keep;
    const long long key_tiles = (keys + T8_KEYS - 1) / T8_KEYS;
    long long best = 0;
    plan.splits = 1;
    for (int k = 1; k <= T8_SPLITS && (k == 1 || (key_tiles >= k && ctas * k <= cmlb_num_sms())); k++) {
        int* fit = &room[cmlb_device_index()][k];
        if (!*fit) *fit = k == 1 ? cmlb_num_sms() : cluster_room((const void*)kern, k, C::kThreads, smem);
        if (*fit < 0) continue;
        const long long waves = (ctas + *fit - 1) / *fit, each = (key_tiles + k - 1) / k, t = waves * (5 + each + (k > 1 ? 2 : 0));
        if (k == 1 || t < best) { best = t; plan.splits = k; }
    }
    CMLB_CUDA(launch_chain(kern, dim3(plan.splits, a->kv_heads * blocks, tiles), dim3(C::kThreads), smem, plan.splits, st, *a, d_qkv, ld, (const int4*)d_tiles, d_out, out_ld, plan, status));
    return CMLB200_OK;
}

}  // namespace

int cmlb_attention8_status_word(int** word) {
    int dev = 0;
    CMLB_CUDA(cudaGetDevice(&dev));
    CMLB_REQUIRE(dev >= 0 && dev < kMaxDevices, "device %d", dev);
    CMLB_CUDA(g_status8.get(dev, word));
    return CMLB200_OK;
}

int cmlb_attention8_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, cudaStream_t st) {
    int* status;
    const int rc = cmlb_attention8_status_word(&status);
    if (rc) return rc;
    if (cmlb_attention8_wide_fits(a, tiles)) return cmlb_attention8_wide(a, d_qkv, ld, d_tiles, tiles, d_out, out_ld, status, st);
    const int widest = a->dim_ld > a->vdim_ld ? a->dim_ld : a->vdim_ld;
#define T8_ARGS a, d_qkv, ld, d_tiles, tiles, d_out, out_ld, status, st
#define T8_FORM(I8, S) return a->slopes ? launch_tiles<I8, S, true>(T8_ARGS) : launch_tiles<I8, S, false>(T8_ARGS)
#define T8_SIZES(I8)                        \
    do {                                    \
        if (widest <= 64) T8_FORM(I8, 1);   \
        if (widest <= 128) T8_FORM(I8, 2);  \
        T8_FORM(I8, 4);                     \
    } while (0)
    if (a->cache_dtype == CMLB200_DT_I8) T8_SIZES(true);
    T8_SIZES(false);
#undef T8_SIZES
#undef T8_FORM
#undef T8_ARGS
}

extern "C" int cmlb200_attention8_status(int* status, int reset) {
    CMLB_REQUIRE(status, "cmlb200_attention8_status: NULL argument");
    int* word;
    const int rc = cmlb_attention8_status_word(&word);
    if (rc) return rc;
    *status = *static_cast<volatile int*>(word);
    if (reset) *static_cast<volatile int*>(word) = 0;
    return CMLB200_OK;
}
