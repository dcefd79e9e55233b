// Pieces of the tcgen05 kernels that attend to 8-bit caches with prompt portions (attention8_tiles.cu, attention8_wide.cu): tiles of up to 64
// rows of one sequence against key tiles of 128 tokens.
#pragma once
#include "cache8.cuh"
#include "pairs.cuh"
#include "tcgen05_util.cuh"

namespace {

constexpr int T8_KEYS = 128, T8_SLAB = T8_KEYS * 128, T8_ROWS = 128, T8_GROUPS = T8_KEYS / kScaleTokens, T8_SPLITS = 8;
constexpr float kLazy = 8.f, kWeightBits = 7.f, kFarScale = -60.f;

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

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
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
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[N][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < N; c++)
#pragma unroll
        for (int j = 0; j < 32; j++) asm volatile("" : "+r"(r[c][j]));
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// registers of a thread are shared out by role, whole warpgroups at a time
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }


// The key tiles of a tile of rows: those of the kept tokens, then from k_lo on (one run from 0 where they meet). A cluster's CTA takes rank, rank + splits, .. Groups from
// hidden_from up to hidden_to lie between the kept tokens and what the first row sees.
struct T8Keys {
    int k_lo, kept_tiles, count, p_last, rank, splits, hidden_from, hidden_to;
    __device__ __forceinline__ T8Keys(const cmlb200_attn& a, int p0, int last, int r, int s) : p_last(last), rank(r), splits(s) {
        k_lo = first_key8(a, p0) & ~(kScaleTokens - 1);
        hidden_from = a.keep;
        hidden_to = k_lo;
        kept_tiles = (min(a.keep, k_lo) + T8_KEYS - 1) / T8_KEYS;
        if (kept_tiles * T8_KEYS >= k_lo) { k_lo = 0; kept_tiles = 0; }
        const int total = kept_tiles + (p_last - k_lo) / T8_KEYS + 1;
        count = rank < total ? (total - rank + splits - 1) / splits : 0;
    }
    __device__ __forceinline__ int start(int i) const { const int t = rank + i * splits; return t < kept_tiles ? t * T8_KEYS : k_lo + (t - kept_tiles) * T8_KEYS; }
};

// Which token and query head of the key/value head a row of the products is: one head's n tokens after the other's, from row `first` on, so that short tiles of
// many heads fill as few rows as they can (13 tokens of 4 heads: 52 of one CTA's 128).
struct T8Rows {
    int n, group, first;
    float per;                                         // 1 / n
    __device__ __forceinline__ T8Rows(int rows, int heads, int first_) : n(max(rows, 1)), group(rows > 0 ? heads : 0), first(first_), per(1.0f / (float)max(rows, 1)) {}
    // whether there is such a row
    __device__ __forceinline__ bool find(int r, int& token, int& h) const {
        h = (int)(((float)(first + r) + 0.5f) * per);  // (exact: two roundings of a number below 2^22 reach no whole one half a row away)
        token = first + r - h * n;
        return h < group;
    }
    __device__ __forceinline__ bool none() const { return first >= n * group; }
};

// The same with 64 rows a head, from head `hb` on: for tiles that are full, and registers that are scarce.
struct T8Heads {
    int n, group, hb;
    __device__ __forceinline__ bool find(int r, int& token, int& h) const {
        h = hb + (r >> 6);
        token = r & 63;
        return token < n && h < group;
    }
};

// Queries into shared memory, each over a power of two of its own (units), in blocks of 128 rows of S slabs. WARPS warps call it, `warp` their number. 8 S lanes
// take a row, 8 numbers each: what they store is one 16-byte piece of the swizzled row. A loop of few instructions with the next row's loads under way: a launch
// begins with cold instruction caches, and six rows at once, unrolled, took longer (64 rows, no cache: 9.4 us, with this 9.3; 2,048: 60.4, with this 56.5).
template <int S, int ROWS, int WARPS, typename Rows>
__device__ __forceinline__ void t8_queries(const cmlb200_attn& a, const float* __restrict__ qkv, int ld, const int4& tl, const Rows& rows, int kh, uint8_t* smem, float* units, int warp) {
    constexpr int kLanes = 8 * S, kStep = WARPS * (32 / kLanes), kEach = (ROWS + kStep - 1) / kStep;
    const int lane = threadIdx.x & 31, d0 = 8 * (lane % kLanes), left = a.dim - d0;
    const float f = a.scale * kLog2e;
    const bool quads = ((reinterpret_cast<uintptr_t>(qkv) & 15) | (unsigned)((ld | a.dim) & 3)) == 0;
    qkv += (size_t)tl.x * ld + (size_t)kh * rows.group * a.dim + d0;
    float x[8], y[8];
    auto fetch = [&](int r) {
        int i, h;
        const bool on = rows.find(r, i, h) && r < ROWS && left > 0;
        const float* src = qkv + (size_t)i * ld + h * a.dim;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = 0.f;
        if (on && quads) {
            const float4 u = *reinterpret_cast<const float4*>(src);
            y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w;
            if (left > 4) {
                const float4 w = *reinterpret_cast<const float4*>(src + 4);
                y[4] = w.x; y[5] = w.y; y[6] = w.z; y[7] = w.w;
            }
        } else if (on) {
#pragma unroll
            for (int e = 0; e < 8; e++) if (e < left) y[e] = src[e];
        }
    };
    int r = warp * (32 / kLanes) + lane / kLanes;
    fetch(r);
#pragma unroll 1
    for (int b = 0; b < kEach; b++, r += kStep) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = y[e] * f;
        fetch(r + kStep);
        uint32_t most = 0;                             // (numbers that are not negative are in order as their bits are)
#pragma unroll
        for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(fabsf(x[e])));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        // a power of two and one over it
        const uint32_t u = most ? max(min(most & 0x7F800000u, 0x7E000000u), 0x00800000u) : 0x3F800000u;
        const float inv = __uint_as_float(0x7F000000u - u);
        if (r >= ROWS) continue;
        if (d0 == 0) units[r] = __uint_as_float(u);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const __half2 t = __floats2half2_rn(x[2 * e] * inv, x[2 * e + 1] * inv);
            w[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(smem + ((r >> 7) * S + (d0 >> 6)) * (T8_ROWS * 128) + (r & 127) * 128 + ((((d0 >> 3) ^ r) & 7) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// What a thread of a team of four warps needs to bring one tile after another of keys or values from the cache into shared memory, as fp16 with 128-byte
// swizzle, S slabs of 64 dimensions. Only this: codes, not scales.
// A slab's 512 pieces of 16 codes: four neighbouring lanes take a key's 64 dimensions, so 64 bytes lie together in a request, and eight lanes' stores,
// of an even key and the odd one behind it, meet all banks. Piece j of a thread: slab j / 4, key tid / 4 + 32 (j % 4), whose group is
// tid / 64 + 2 (j % 4); a batch is kept in registers.
template <bool I8, int S, int BATCH>
struct T8Team {
    static constexpr int BATCHES = 4 * S / BATCH;
    const uint8_t* base;
    int stride, width, c16, in_group, g0;
    uint32_t to, even;
    uint4 u[BATCH];
    __device__ __forceinline__ void init(const void* pool, int kh, int kv_heads, int w, uint32_t smem, int tid) {
        width = w;
        c16 = 16 * (tid & 3);
        in_group = (tid >> 2) & 15;
        g0 = tid >> 6;
        base = static_cast<const uint8_t*>(pool) + (size_t)kh * width + c16;
        stride = kv_heads * width;
        to = smem + (tid >> 2) * 128;
        even = ((2 * (tid & 3)) ^ ((tid >> 2) & 7)) << 4;
    }
    // tok: the thread's four keys
    __device__ __forceinline__ void load(const int (&tok)[4], int batch) {
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            const int d = 64 * ((batch * BATCH + j) >> 2);
            u[j] = make_uint4(0u, 0u, 0u, 0u);
            if (d + c16 < width) u[j] = *reinterpret_cast<const uint4*>(base + (size_t)tok[j & 3] * stride + d);
        }
    }
    __device__ __forceinline__ void store(int stage_at, int batch) const {
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            const int slab = (batch * BATCH + j) >> 2;
            if (64 * slab + c16 >= width) continue;
            uint32_t h[8];
            unpack8<I8>(u[j].x, h[0], h[1]);
            unpack8<I8>(u[j].y, h[2], h[3]);
            unpack8<I8>(u[j].z, h[4], h[5]);
            unpack8<I8>(u[j].w, h[6], h[7]);
            const uint32_t at = to + stage_at + slab * T8_SLAB + 32 * 128 * (j & 3);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + even), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + (even ^ 16)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
        }
    }
    // all of a tile whose first batch is in registers
    __device__ __forceinline__ void store_tile(const int (&tok)[4], int stage_at) {
        store(stage_at, 0);
#pragma unroll
        for (int b = 1; b < BATCHES; b++) {
            load(tok, b);
            store(stage_at, b);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
};
// A tile's scales as the softmax finds them: 8 key scales, log2 of 8 value scales; four tiles in turn.
constexpr int T8_SCALES = 2 * T8_GROUPS;
struct T8Scaler {
    bool on;                                           // lanes 0 .. 7 of one warp look after key scales, 8 .. 15 after value scales
    int lane, kh;
    float scale;
    __device__ __forceinline__ void fetch(const cmlb200_attn& a, int token) {
        if (on) scale = (lane < T8_GROUPS ? a.k_scale : a.v_scale)[(size_t)token / kScaleTokens * a.kv_heads + kh];
    }
    __device__ __forceinline__ void put(float* scales, int i) const {
        if (on) scales[(i & 3) * T8_SCALES + lane] = lane < T8_GROUPS ? scale : log2f(fmaxf(scale, 1.17549435e-38f));
    }
};
// Where group `lane & 7` of tile i begins in the pools; groups behind the last row's are read as that one, and those behind the kept tokens that no row sees as the first: their pages
// may be anybody's by now.
__device__ __forceinline__ int t8_place(const cmlb200_attn& a, const int* table, int shift, const T8Keys& keys, int i, int lane) {
    int first = min(keys.start(i) + kScaleTokens * (lane & 7), keys.p_last & ~(kScaleTokens - 1));
    if (first >= keys.hidden_from && first < keys.hidden_to) first = 0;
    return (table[first >> shift] << shift) + (first & (a.block_size - 1));
}
// A thread's four keys of the tile whose groups lie at `at` (t8_place); keys behind the last row are read as that one.
__device__ __forceinline__ void t8_tokens(int (&tok)[4], int at, int kt, int p_last, int g0, int in_group) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int g = g0 + 2 * j, rest = p_last - kt - 16 * g;
        tok[j] = __shfl_sync(0xffffffffu, at, g) + (rest < 0 ? p_last & (kScaleTokens - 1) : min(in_group, rest));
    }
}

// Columns 16 e .. 16 e + 15 of 32 scores, all of one group with the factor f; j0: the first one's place among the thread's keys. Their largest, in units of log2
// without the bias that all of the thread's keys share.
template <bool SLOPES>
__device__ __forceinline__ float t8_group_max(const uint32_t (&v)[32], int e, float f, float slope, int j0) {
    auto x = [&](int j) { const float y = __uint_as_float(v[16 * e + j]); return SLOPES ? fmaf(y, f, slope * (float)(j0 + j)) : y; };
    float t0 = x(0), t1 = x(1);
#pragma unroll
    for (int j = 2; j < 14; j += 4) { t0 = max3(t0, x(j), x(j + 1)); t1 = max3(t1, x(j + 2), x(j + 3)); }
    t0 = fmaxf(max3(t0, x(14), x(15)), t1);
    return SLOPES ? t0 : t0 * f;
}
// Their weights 2^(score + b) as pairs of fp16 into w[8 e ..]; the sum of them.
template <bool SLOPES>
__device__ __forceinline__ float t8_group_weights(const uint32_t (&v)[32], uint32_t (&w)[16], int e, float f, float b, float slope, int j0) {
    const uint64_t ff = pair_of(f, f), bb = pair_of(b, b), sl = pair_of(slope, slope);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int k = 16 * e + 2 * j;
        uint64_t y = fma_pair(pair_of(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), ff, bb);
        if (SLOPES) y = fma_pair(sl, pair_of((float)(j0 + 2 * j), (float)(j0 + 2 * j + 1)), y);
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
    return t0 + t1;
}
// O's columns c0, c0 + step, .. (16 each) times c
__device__ __forceinline__ void t8_scale_o(uint32_t o_at, int c0, int step, int dv, float c) {
#pragma unroll 1
    for (; c0 < dv; c0 += step) {
        uint32_t o[16];
        tmem_ld16(o_at + c0, o);
#pragma unroll
        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * c);
        tmem_st16(o_at + c0, o);
    }
}

// A row's columns c0, c0 + step, .. (32 each) of O, times inv and its gates, into the output. live: there is such a row. The whole warp calls it.
__device__ __forceinline__ void t8_write_row(const cmlb200_attn& a, uint32_t o_at, int c0, int step, bool live, float inv, const float* row, int head, __nv_bfloat16* out, int out_ld, size_t at) {
    const int dv = a.vdim_ld;
    __nv_bfloat16* dst = out + at * out_ld + (size_t)head * a.vdim;
    const bool wide = ((reinterpret_cast<uintptr_t>(out) | (unsigned)(out_ld * 2) | (unsigned)(a.vdim * 2)) & 15) == 0;
#pragma unroll 1
    for (; c0 < dv; c0 += step) {
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
}

}  // namespace

// attention8_wide.cu. _fits: 1 where that form is the faster one
bool cmlb_attention8_wide_fits(const cmlb200_attn* a, int tiles);
int cmlb_attention8_wide(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_tiles, int tiles, __nv_bfloat16* d_out, int out_ld, int* status, cudaStream_t st);
