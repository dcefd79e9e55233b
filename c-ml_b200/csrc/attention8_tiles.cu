// Prompt portions over 8-bit caches (cache8.cuh) on the 5th-generation tensor cores.
//
// A CTA takes a tile of up to 64 consecutive rows of one sequence and 2 NM query heads of a key/value head: NM blocks of 128 rows (64 tokens x 2
// heads) that share the expansion of the codes. Key tiles of 128 tokens; S = Q K^T, and O += P V with P in tensor memory over the scores it came from.
// Tensor memory: per block 128 columns of scores, then 128 (256 for wider values) of output. Roles, by warp:
//   0 .. 4 NM - 1   softmax, a thread a row: the largest score of the tile, then exponentials straight into P, 32 columns at a time. The reference of the
//                   exponentials moves, and O is scaled, only when a row has grown by more than 8 (powers of two)
//   next 4          expansion: codes from the cache (the next tile's are requested before this one's are written) to fp16 in shared memory, keys with
//                   the dimensions contiguous, values with theirs as the contiguous non-summed side, both with 128-byte swizzle. Codes are exact
//                   in fp16; scales stay apart: a group's key scale multiplies its scores, its value scale joins the exponent of its weights
//   last            issues tcgen05.mma, block by block: P V of a tile, then the scores of the next. While one block's softmax runs the other's products do;
//                   products are done in order, so that a block's scores being there means that its O is at rest too
// Queries are fp16 over a power of two per row and head. Weights are 2^(s - m) times the value scale over the largest so far, times 128: at most 2^15.
// Few tiles: a cluster of up to 8 CTAs splits the keys and merges through distributed shared memory.
// Keys behind a portion's last row are read as that row's (their weights are zero), so nothing other requests left can reach the sums. Every wait is
// bounded; one that gives up leaves a code in a status word in host memory, the products under way are waited for and tensor memory is freed.
#include "cache8.cuh"
#include "tcgen05_util.cuh"

namespace {

constexpr int T8_KEYS = 128, T8_SLAB = T8_KEYS * 128, T8_ROWS = 128, T8_GROUPS = T8_KEYS / kScaleTokens, T8_SPLITS = 8;
constexpr float kLazy = 8.f, kWeightBits = 7.f, kFarScale = -60.f;

__device__ __forceinline__ int first_key8(const cmlb200_attn& a, int p) {
    if (a.chunk > 0) return p / a.chunk * a.chunk;
    return (a.window > 0 && a.window <= p) ? p - a.window + 1 : 0;
}
// Products whose descriptors differ from one another in their lower halves alone.
__device__ __forceinline__ void umma_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n"
                 ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accum) : "memory");
}
// A from tensor memory: 128 rows of 16 fp16 numbers in 8 columns
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n"
                 ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}

// Shared memory of a CTA: queries, key stages, value stages, then the small things.
// two numbers at a time
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void tmem_ld32_begin(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// nothing that reads the registers moves ahead of this
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[4][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int j = 0; j < 32; j++) asm volatile("" : "+r"(r[c][j]));
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct T8Plan {
    int stages;                                        // of keys and of values
    int splits;
};
template <int NM, int SK, int SV>
struct T8 {
    static constexpr int kThreads = 32 * (4 * NM + 8), kSoft = 128 * NM;
    // registers of a thread: 128 and 168 at launch, then shared out (176 x 256 + 104 x 128 + 56 x 128 = 128 x 512; 232 + 168 + 56 < 3 x 168)
    static constexpr int kSoftRegs = NM == 2 ? 176 : 232, kConvRegs = NM == 2 ? 104 : 168, kIssueRegs = 56;
    static constexpr int kQ = NM * SK * T8_ROWS * 128, kK = SK * T8_SLAB, kV = SV * T8_SLAB;
    static constexpr int kCols = NM * 128 + NM * SV * 64;                     // tensor memory
    static constexpr int kTmem = kCols <= 256 ? 256 : 512;
    static constexpr int kSmall = 2048 + 3 * 4 * NM * T8_ROWS;
    static int bytes(int stages) { return 1024 + kQ + stages * (kK + kV) + kSmall; }
};

// grid = (splits, kv_heads * blocks, tiles), clusters of `splits`; SK, SV: slabs of 64 dimensions of a key and a value.
template <bool I8, int NM, int SK, int SV, bool SLOPES>
__global__ void __launch_bounds__(T8<NM, SK, SV>::kThreads, 1)
attention8_tiles_kernel(const cmlb200_attn a, const float* __restrict__ qkv, int ld, const int4* __restrict__ tiles, __nv_bfloat16* __restrict__ out, int out_ld, const T8Plan plan,
                        int* status) {
    using C = T8<NM, SK, SV>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const int dk = a.dim_ld, dv = a.vdim_ld, stages = plan.stages, splits = plan.splits, rank = blockIdx.x;
    uint8_t* small = smem + C::kQ + stages * (C::kK + C::kV);
    const uint32_t qs = smem_addr(smem), ks = qs + C::kQ, vs = ks + stages * C::kK, bars = smem_addr(small);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto s_full = [&](int m) { return bars + 64 + 8 * m; };
    auto p_full = [&](int m) { return bars + 80 + 8 * m; };
    auto o_full = [&](int m) { return bars + 96 + 8 * m; };
    const uint32_t drained = bars + 112;
    auto p_more = [&](int m) { return bars + 120 + 8 * m; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(small + 144);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(small + 152);
    float* scales = reinterpret_cast<float*>(small + 256);                    // [4 stages][2][T8_GROUPS]: key scales, log2 of value scales (tile i in i & 3)
    float* unit_s = reinterpret_cast<float*>(small + 2048);                   // [NM * 128] powers of two of the queries; then maxima and sums
    float* c_m = unit_s + NM * T8_ROWS;
    float* c_l = c_m + NM * T8_ROWS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConv = 4 * NM, kIssue = 4 * NM + 4;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) { mbar_init(k_full(s), 4); mbar_init(k_empty(s), 1); mbar_init(v_full(s), 4); mbar_init(v_empty(s), 1); }
        for (int m = 0; m < 2; m++) { mbar_init(s_full(m), 1); mbar_init(p_full(m), 4); mbar_init(p_more(m), 4); mbar_init(o_full(m), 1); }
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((uint32_t)C::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dep_wait();
    const int4 tl = tiles[gridDim.z - 1 - blockIdx.z];                       // a prompt's last tiles, which see most keys, come first
    const int group = a.heads / a.kv_heads, blocks = gridDim.y / a.kv_heads, kh = blockIdx.y / blocks, hb = blockIdx.y % blocks * 2 * NM;
    const int n = tl.y, p0 = tl.w, p_last = p0 + n - 1, shift = __ffs(a.block_size) - 1;
    const int* table = a.block_table + (size_t)tl.z * a.table_ld;
    // key tiles: those of the kept tokens, then from k_lo on (one run from 0 where they meet)
    int k_lo = first_key8(a, p0) & ~(kScaleTokens - 1), kept_tiles = (min(a.keep, k_lo) + T8_KEYS - 1) / T8_KEYS;
    if (kept_tiles * T8_KEYS >= k_lo) { k_lo = 0; kept_tiles = 0; }
    const int total = kept_tiles + (p_last - k_lo) / T8_KEYS + 1, count = rank < total ? (total - rank + splits - 1) / splits : 0;      // of this CTA: rank, rank + splits, ..
    auto tile_start = [&](int i) { const int t = rank + i * splits; return t < kept_tiles ? t * T8_KEYS : k_lo + (t - kept_tiles) * T8_KEYS; };

    // ---- the queries: row 64 h + i of block m is token i of head hb + 2 m + h, over a power of two of its own
    if (count > 0) {
        const float f = a.scale * kLog2e;
        constexpr int kAhead = 16 / SK, kWarps = C::kThreads / 32;            // rows whose loads are under way together
        for (int r0 = warp; r0 < NM * T8_ROWS; r0 += kAhead * kWarps) {
            float2 x[kAhead][SK];
#pragma unroll
            for (int b = 0; b < kAhead; b++) {
                const int r = r0 + b * kWarps, i = r & 63, h = hb + (r >> 6);
                const bool live = r < NM * T8_ROWS && i < n && h < group;
                const float* src = qkv + (size_t)(tl.x + (live ? i : 0)) * ld + (size_t)(kh * group + (live ? h : 0)) * a.dim;
#pragma unroll
                for (int s = 0; s < SK; s++) {
                    const int d = 64 * s + 2 * lane;
                    x[b][s].x = live && d < a.dim ? src[d] : 0.f;
                    x[b][s].y = live && d + 1 < a.dim ? src[d + 1] : 0.f;
                }
            }
#pragma unroll
            for (int b = 0; b < kAhead; b++) {
                const int r = r0 + b * kWarps;
                if (r >= NM * T8_ROWS) break;
                float most = 0.f;
#pragma unroll
                for (int s = 0; s < SK; s++) { x[b][s].x *= f; x[b][s].y *= f; most = fmaxf(most, fmaxf(fabsf(x[b][s].x), fabsf(x[b][s].y))); }
                most = lane_max(most);
                const float unit = most > 0.f ? __uint_as_float(max(min(__float_as_uint(most) & 0x7F800000u, 0x7E000000u), 0x00800000u)) : 1.0f, inv = 1.0f / unit;
                if (lane == 0) unit_s[r] = unit;
                uint8_t* dst = smem + (r >> 7) * (SK * T8_ROWS * 128) + (r & 127) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
#pragma unroll
                for (int s = 0; s < SK; s++) *reinterpret_cast<__half2*>(dst + s * (T8_ROWS * 128)) = __floats2half2_rn(x[b][s].x * inv, x[b][s].y * inv);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    dep_trigger();                                     // a launch that allocates tensor memory too may start from here on: every CTA of this one has its own

    if (warp < kConv) {                                // ---- softmax
        more_registers<C::kSoftRegs>();
        const int m = warp >> 2, r = (warp & 3) * 32 + lane, i_tok = r & 63, h = hb + 2 * m + (r >> 6);
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_at = lanes + m * 128, o_at = lanes + NM * 128 + m * (SV * 64);
        const bool live = i_tok < n && h < group;
        // (rows that are none have queries of zero and see what the last one sees; nobody looks at theirs)
        const int p = live ? p0 + i_tok : p_last, lo = first_key8(a, p), lo_last = first_key8(a, p_last), head = kh * group + (live ? h : 0);
        const float unit = unit_s[m * T8_ROWS + r], slope = SLOPES && live ? a.slopes[head] * kLog2e : 0.f;
        float mx_ref = -INFINITY, l = 0.f, vref = -INFINITY;
        bool ok = true;
        for (int i = 0; i < count; i++) {
            const int kt = tile_start(i);
            ok = __all_sync(0xffffffffu, mbar_wait(s_full(m), i & 1, abort_flag, 1, status));
            if (!ok) break;
            tmem_fence_after();
            uint32_t v[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32_begin(s_at + 32 * c, v[c]);
            const float* sc = scales + (i & 3) * 2 * T8_GROUPS;
            float vm = vref;
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
            float mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < T8_GROUPS; g++) {
                const float f = factor(g);
                auto x = [&](int j) { const float y = __uint_as_float(v[g >> 1][16 * (g & 1) + j]); return SLOPES ? fmaf(y, f, slope * (float)(16 * g + j)) : y; };
                float t0 = x(0), t1 = x(1);
#pragma unroll
                for (int j = 2; j < 14; j += 4) { t0 = max3(t0, x(j), x(j + 1)); t1 = max3(t1, x(j + 2), x(j + 3)); }
                t0 = fmaxf(max3(t0, x(14), x(15)), t1);
                mx = fmaxf(mx, SLOPES ? t0 : t0 * f);
            }
            mx += far;
            if (__any_sync(0xffffffffu, mx > mx_ref + kLazy || vm > vref)) {
                const float nm = fmaxf(mx_ref, mx), c = nm == -INFINITY ? 1.f : ex2(mx_ref - nm), cv = ex2(vref - vm);
                mx_ref = nm;
                vref = vm;
                l *= c;
                if (i > 0) {
#pragma unroll 1
                    for (int c0 = 0; c0 < dv; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_at + c0, o);
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * (c * cv));
                        tmem_st16(o_at + c0, o);
                    }
                }
            }
            const float u = (mx_ref == -INFINITY ? 0.f : mx_ref) - far;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int g = 2 * c + e;
                    const float f = factor(g), bits = fmaxf(sc[T8_GROUPS + g] - vref, kFarScale) + kWeightBits, b = bits - u;
                    const uint64_t ff = pair_of(f, f), bb = pair_of(b, b), sl = pair_of(slope, slope);
                    uint64_t sum = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int k = 16 * e + 2 * j;
                        uint64_t y = fma_pair(pair_of(__uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1])), ff, bb);
                        if (SLOPES) y = fma_pair(sl, pair_of((float)(32 * c + k), (float)(32 * c + k + 1)), y);
                        float e0, e1;
                        unpair(y, e0, e1);
                        e0 = ex2(e0);
                        e1 = ex2(e1);
                        sum = add_pair(sum, pair_of(e0, e1));
                        const __half2 x = __floats2half2_rn(e0, e1);
                        w[8 * e + j] = *reinterpret_cast<const uint32_t*>(&x);
                    }
                    float t0, t1;
                    unpair(sum, t0, t1);
                    l = fmaf(t0 + t1, ex2(-bits), l);
                }
                tmem_st16(s_at + 16 * c, w);           // over the scores, which are all in registers
                if (c & 1) {                           // half of the tile's keys: their product may begin
                    tmem_st_wait();
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(c == 1 ? p_full(m) : p_more(m));
                }
            }
        }
        if (ok && count > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_full(m), 0, abort_flag, 2, status));
        tmem_fence_after();
        const float back = count > 0 && ok ? ex2(vref - kWeightBits) : 0.f;
        const float* row = qkv + (size_t)(tl.x + (live ? i_tok : 0)) * ld;
        if (splits == 1) {
            float all = l;
            if (a.sink && l > 0.f) all += ex2((a.sinks ? a.sinks[head] : 0.f) * kLog2e - mx_ref);
            float inv = ok && all > 0.f ? back * (a.out_scale == 0.f ? 1.f : a.out_scale) / all : 0.f;
            if (a.gate_col >= 0 && !a.gate_wide && live) inv *= sigmoidf(row[a.gate_col + head]);
            __nv_bfloat16* dst = out + (size_t)(tl.x + (live ? i_tok : 0)) * out_ld + (size_t)head * a.vdim;
            const bool wide = ((reinterpret_cast<uintptr_t>(out) | (unsigned)(out_ld * 2) | (unsigned)(a.vdim * 2)) & 15) == 0;
#pragma unroll 1
            for (int c0 = 0; c0 < dv; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + c0, o);
                if (live && a.gate_wide) {
                    const float* gate = row + a.gate_col + head * a.vdim + c0;
#pragma unroll
                    for (int j = 0; j < 32; j++) if (c0 + j < a.vdim) o[j] = __float_as_uint(__uint_as_float(o[j]) * sigmoidf(gate[j]));
                }
                if (live && wide && c0 + 32 <= a.vdim) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv);
                        w[j] = *reinterpret_cast<const uint32_t*>(&b);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) *reinterpret_cast<uint4*>(dst + c0 + 8 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                } else if (live) {
#pragma unroll
                    for (int j = 0; j < 32; j++) if (c0 + j < a.vdim) dst[c0 + j] = __float2bfloat16_rn(__uint_as_float(o[j]) * inv);
                }
                __syncwarp();
            }
        } else {
            // nothing of this CTA's operands is needed any more: all of the products are done once both blocks' are
            if (NM == 2 && ok && count > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_full(m ^ 1), 0, abort_flag, 3, status));
            c_m[m * T8_ROWS + r] = ok ? mx_ref : -INFINITY;
            c_l[m * T8_ROWS + r] = ok ? l : 0.f;
            float* Os = reinterpret_cast<float*>(smem) + (size_t)(m * T8_ROWS + r) * (dv + 4);
#pragma unroll 1
            for (int c0 = 0; c0 < dv && count > 0 && ok; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + c0, o);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c0 + 4 * j < dv)
                        *reinterpret_cast<float4*>(Os + c0 + 4 * j) = make_float4(__uint_as_float(o[4 * j]) * back, __uint_as_float(o[4 * j + 1]) * back, __uint_as_float(o[4 * j + 2]) * back, __uint_as_float(o[4 * j + 3]) * back);
            }
        }
        tmem_fence_before();
        __syncwarp();
        if (splits > 1) {
            cluster_meet();
            const int quads = dv / 4, width = dv + 4;
            for (int e = rank * C::kSoft + threadIdx.x; e < NM * T8_ROWS * quads; e += splits * C::kSoft) {
                const int r = e / quads, c = (e - r * quads) * 4, i = r & 63, h = hb + (r >> 6);
                if (i >= n || h >= group) continue;
                float ms[T8_SPLITS], ls[T8_SPLITS], mx = -INFINITY;
    #pragma unroll
                for (int s = 0; s < T8_SPLITS; s++) {
                    ms[s] = -INFINITY;
                    ls[s] = 0.f;
                    if (s < splits) {
                        uint32_t am, al;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(am) : "r"(smem_addr(c_m + r)), "r"(s));
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(al) : "r"(smem_addr(c_l + r)), "r"(s));
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ms[s]) : "r"(am) : "memory");
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ls[s]) : "r"(al) : "memory");
                    }
                    mx = fmaxf(mx, ms[s]);
                }
                const int head = kh * group + h;
                float sum = 0.f;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    #pragma unroll
                for (int s = 0; s < T8_SPLITS; s++) {
                    if (s >= splits || ms[s] == -INFINITY) continue;             // saw nothing: its values may be anything
                    uint32_t ax;
                    float4 y;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ax) : "r"(smem_addr(reinterpret_cast<float*>(smem) + (size_t)r * width + c)), "r"(s));
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(ax) : "memory");
                    const float f = exp2f(ms[s] - mx);
                    sum = fmaf(ls[s], f, sum);
                    x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
                }
                if (a.sink && sum > 0.f) sum += exp2f((a.sinks ? a.sinks[head] : 0.f) * kLog2e - mx);
                float inv = sum > 0.f ? (a.out_scale == 0.f ? 1.f : a.out_scale) / sum : 0.f;
                const float* row = qkv + (size_t)(tl.x + i) * ld;
                if (a.gate_col >= 0 && !a.gate_wide) inv *= sigmoidf(row[a.gate_col + head]);
                const float v[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
                __nv_bfloat16* dst = out + (size_t)(tl.x + i) * out_ld + (size_t)head * a.vdim;
    #pragma unroll
                for (int j = 0; j < 4; j++)
                    if (c + j < a.vdim) dst[c + j] = __float2bfloat16_rn(a.gate_wide ? v[j] * sigmoidf(row[a.gate_col + head * a.vdim + c + j]) : v[j]);
            }
            __syncwarp();
            cluster_meet();                            // nobody leaves while others read its shared memory
        }
    } else if (warp < kIssue) {                        // ---- expansion
        if (NM == 2) fewer_registers<C::kConvRegs>();
        const int tid = threadIdx.x - kConv * 32, w4 = warp - kConv;
        // A slab's 512 pieces of 16 codes: four neighbouring lanes take a key's 64 dimensions, so 64 bytes lie together in a request, and eight lanes' stores,
        // of an even key and the odd one behind it, meet all banks. Piece j of a thread: slab j / 4, key tid / 4 + 32 (j % 4); a batch is kept in registers.
        constexpr int BATCH = SK == 1 ? 4 : 8, KB = 4 * SK / BATCH, VB = 4 * SV / BATCH;
        static_assert(SK == SV, "batches are alike");
        const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + (size_t)kh * dk;
        const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + (size_t)kh * dv;
        const size_t kstride = (size_t)a.kv_heads * dk, vstride = (size_t)a.kv_heads * dv;
        // lane g of a warp knows where group g & 7 of a tile begins, keys behind the last row end with it
        auto place = [&](int i) {
            const int key = min(tile_start(i) + kScaleTokens * (lane & 7), p_last & ~(kScaleTokens - 1));
            return (table[key >> shift] << shift) + (key & (a.block_size - 1));
        };
        auto token_of = [&](int at, int kt, int row) {
            const int g = row >> 4, first = __shfl_sync(0xffffffffu, at, g), rest = p_last - kt - 16 * g;      // rows of the group that exist, less one
            return (size_t)first + (rest < 0 ? p_last & (kScaleTokens - 1) : min(row & 15, rest));
        };
        const int c16 = 16 * (tid & 3);
        auto load = [&](uint4 (&u)[BATCH], int at, int kt, const uint8_t* base, size_t stride, int width, int batch) {
#pragma unroll
            for (int j = 0; j < BATCH; j++) {
                const int row = (tid >> 2) + 32 * (j & 3), d = 64 * ((batch * BATCH + j) >> 2) + c16;
                const size_t token = token_of(at, kt, row);
                u[j] = make_uint4(0u, 0u, 0u, 0u);
                if (d < width) u[j] = *reinterpret_cast<const uint4*>(base + token * stride + d);
            }
        };
        auto store = [&](const uint4 (&u)[BATCH], uint32_t dst, int width, int batch) {
#pragma unroll
            for (int j = 0; j < BATCH; j++) {
                const int row = (tid >> 2) + 32 * (j & 3), slab = (batch * BATCH + j) >> 2;
                if (64 * slab + c16 >= width) continue;
                uint32_t h[8];
                unpack8<I8>(u[j].x, h[0], h[1]);
                unpack8<I8>(u[j].y, h[2], h[3]);
                unpack8<I8>(u[j].z, h[4], h[5]);
                unpack8<I8>(u[j].w, h[6], h[7]);
                const uint32_t at = dst + slab * T8_SLAB + row * 128, a0 = at + (((2 * (tid & 3)) ^ (row & 7)) << 4), a1 = at + (((2 * (tid & 3) + 1) ^ (row & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a1), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
            }
        };
        bool ok = true;
        int st = 0, par = 1, at = 0;
        uint4 ku[BATCH], vu[BATCH];
        if (count > 0) {
            at = place(0);
            load(ku, at, tile_start(0), kp, kstride, dk, 0);
            load(vu, at, tile_start(0), vp, vstride, dv, 0);
        }
        for (int i = 0; i < count; i++) {
            const int kt = tile_start(i), more = i + 1 < count, next = more ? place(i + 1) : 0, kn = more ? tile_start(i + 1) : 0;
            ok = __all_sync(0xffffffffu, mbar_wait(k_empty(st), par, abort_flag, 4, status));
            if (!ok) break;
            if (w4 == 0 && lane < 2 * T8_GROUPS) {     // (whoever read tile i - 4's has let go of its stage twice over)
                const size_t sc = (size_t)at / kScaleTokens * a.kv_heads + kh;
                scales[(i & 3) * 2 * T8_GROUPS + lane] = lane < T8_GROUPS ? a.k_scale[sc] : log2f(fmaxf(a.v_scale[sc], 1.17549435e-38f));
            }
            store(ku, ks + st * C::kK, dk, 0);
#pragma unroll
            for (int b = 1; b < KB; b++) {
                load(ku, at, kt, kp, kstride, dk, b);
                store(ku, ks + st * C::kK, dk, b);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full(st));
            if (more) load(ku, next, kn, kp, kstride, dk, 0);
            ok = __all_sync(0xffffffffu, mbar_wait(v_empty(st), par, abort_flag, 5, status));
            if (!ok) break;
            store(vu, vs + st * C::kV, dv, 0);
#pragma unroll
            for (int b = 1; b < VB; b++) {
                load(vu, at, kt, vp, vstride, dv, b);
                store(vu, vs + st * C::kV, dv, b);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(st));
            if (more) load(vu, next, kn, vp, vstride, dv, 0);
            at = next;
            if (++st == stages) { st = 0; par ^= 1; }
        }
        __syncwarp();
        if (splits > 1) { cluster_meet(); cluster_meet(); }
    } else {                                           // ---- products
        fewer_registers<C::kIssueRegs>();
        if (warp == kIssue && count > 0) {
            // fp16 operands, fp32 accumulators, 128 rows; the second one takes V with its columns contiguous
            const uint32_t is = (1u << 4) | ((uint32_t)(T8_KEYS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t io = (1u << 4) | (1u << 16) | ((uint32_t)(dv >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int steps = dk >> 4;
            bool ok = true;
            auto scores = [&](int m, int st) {
                if (elect_one()) {
                    const uint64_t ad = make_desc(qs + m * (SK * T8_ROWS * 128)), bd = make_desc(ks + st * C::kK);
                    const uint32_t alo = (uint32_t)ad, blo = (uint32_t)bd, hi = (uint32_t)(ad >> 32);
#pragma unroll
                    for (int k = 0; k < 4 * SK; k++)
                        if (k < steps) umma_lo(tm + m * 128, alo + (k >> 2) * (T8_ROWS * 128 >> 4) + 2 * (k & 3), blo + (k >> 2) * (T8_SLAB >> 4) + 2 * (k & 3), hi, is, k ? 1u : 0u);
                    if (m == NM - 1) umma_commit(k_empty(st));
                    umma_commit(s_full(m));
                }
                __syncwarp();
            };
            int kst = 0, kpar = 0, vst = 0, vpar = 0;
            auto keys = [&]() {
                const bool got = __all_sync(0xffffffffu, mbar_wait(k_full(kst), kpar, abort_flag, 6, status));
                tmem_fence_after();
                return got;
            };
            ok = keys();
            if (ok)
                for (int m = 0; m < NM; m++) scores(m, kst);
            if (++kst == stages) { kst = 0; kpar ^= 1; }
            for (int i = 0; i < count && ok; i++) {
                ok = __all_sync(0xffffffffu, mbar_wait(v_full(vst), vpar, abort_flag, 7, status));
                if (!ok) break;
                for (int m = 0; m < NM && ok; m++) {
                    const uint64_t vd = make_desc_mn(vs + vst * C::kV, T8_SLAB);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(half ? p_more(m) : p_full(m), i & 1, abort_flag, 8, status));
                        if (!ok) break;
                        tmem_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; k++)
                                umma_ts(tm + NM * 128 + m * (SV * 64), tm + m * 128 + 8 * k, (uint32_t)vd + k * (2048 >> 4), (uint32_t)(vd >> 32), io, (i | k) ? 1u : 0u);
                            if (half && m == NM - 1) umma_commit(v_empty(vst));
                            if (half && i + 1 == count) umma_commit(o_full(m));
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (i + 1 < count) {
                        if (m == 0) ok = keys();
                        if (ok) scores(m, kst);
                    }
                }
                if (++vst == stages) { vst = 0; vpar ^= 1; }
                if (++kst == stages) { kst = 0; kpar ^= 1; }
            }
            // nothing that was issued outlives the CTA's tensor memory
            if (elect_one()) umma_commit(drained);
            __syncwarp();
            for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(drained, 0); it++) {}
            __syncwarp();
        }
        __syncwarp();
        if (splits > 1) { cluster_meet(); cluster_meet(); }
    }
    __syncthreads();
    if (warp == kIssue) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmem) : "memory");
    }
}

int* g_status8[kMaxDevices] = {};

int status_word8(int** word) {
    int dev = 0;
    CMLB_CUDA(cudaGetDevice(&dev));
    CMLB_REQUIRE(dev >= 0 && dev < kMaxDevices, "device %d", dev);
    if (!g_status8[dev]) {
        void* p = nullptr;
        CMLB_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocDefault));
        *static_cast<int*>(p) = 0;
        g_status8[dev] = static_cast<int*>(p);
    }
    *word = g_status8[dev];
    return CMLB200_OK;
}

template <bool I8, int NM, int SK, int SV, bool SLOPES>
int launch_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, int* status, cudaStream_t st) {
    using C = T8<NM, SK, SV>;
    const int group = a->heads / a->kv_heads, blocks = (group + 2 * NM - 1) / (2 * NM);
    CMLB_REQUIRE((long long)a->kv_heads * blocks <= 65535 && tiles <= 65535, "cmlb200_attention_tiles: %d tiles, %d heads", tiles, a->heads);
    T8Plan plan;
    for (plan.stages = 2; plan.stages > 1 && C::bytes(plan.stages) > 227 * 1024; plan.stages--) {}
    // few tiles: a cluster shares the keys of each, as far as SMs and keys go (a block table's row holds no more than table_ld blocks)
    const long long ctas = (long long)tiles * a->kv_heads * blocks, reach = a->chunk > 0 ? a->chunk + 64 : a->window > 0 ? a->window + 64 : 0;
    long long keys = (long long)a->table_ld * a->block_size;
    if (reach && reach + a->keep < keys) keys = reach + a->keep;
    for (plan.splits = 1; plan.splits < T8_SPLITS && ctas * plan.splits * 2 <= cmlb_num_sms() && keys > plan.splits * T8_KEYS; plan.splits *= 2) {}
    size_t smem = (size_t)C::bytes(plan.stages);
    // a cluster's CTAs wait for one another while they hold tensor memory: such a CTA has its SM to itself
    if (plan.splits > 1 && smem < 118 * 1024) smem = 118 * 1024;
    static size_t attr[kMaxDevices] = {};
    auto kern = attention8_tiles_kernel<I8, NM, SK, SV, SLOPES>;
    CMLB_CUDA(cmlb_ensure_smem(kern, smem, attr));
    CMLB_CUDA(launch_chain(kern, dim3(plan.splits, a->kv_heads * blocks, tiles), dim3(C::kThreads), smem, plan.splits, st, *a, d_qkv, ld, (const int4*)d_tiles, d_out, out_ld, plan, status));
    return CMLB200_OK;
}

}  // namespace

int cmlb_attention8_tiles(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, cudaStream_t st) {
    int* status;
    const int rc = status_word8(&status);
    if (rc) return rc;
    const int group = a->heads / a->kv_heads, widest = a->dim_ld > a->vdim_ld ? a->dim_ld : a->vdim_ld;
    // two blocks share the expansion where a key/value head has four query heads for them and there are CTAs enough for the SMs
    const bool two = widest <= 128 && group > 2 && (long long)tiles * a->kv_heads * ((group + 3) / 4) >= cmlb_num_sms();
#define T8_ARGS a, d_qkv, ld, d_tiles, tiles, d_out, out_ld, status, st
#define T8_FORM(I8, NM, S) return a->slopes ? launch_tiles<I8, NM, S, S, true>(T8_ARGS) : launch_tiles<I8, NM, S, S, false>(T8_ARGS)
#define T8_SIZES(I8)                        \
    do {                                    \
        if (widest <= 64) {                 \
            if (two) T8_FORM(I8, 2, 1);     \
            T8_FORM(I8, 1, 1);              \
        }                                   \
        if (widest <= 128) {                \
            if (two) T8_FORM(I8, 2, 2);     \
            T8_FORM(I8, 1, 2);              \
        }                                   \
        T8_FORM(I8, 1, 4);                  \
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
    const int rc = status_word8(&word);
    if (rc) return rc;
    *status = *static_cast<volatile int*>(word);
    if (reset) *static_cast<volatile int*>(word) = 0;
    return CMLB200_OK;
}
