// Decoded tokens over 8-bit caches (cache8.cuh), one row per sequence: norm, rotation, append, attention and gate in one launch.
//
// A step reads every cached byte of its sequences once, so HBM bounds it; codes have to become MMA operands in few instructions. A warp
// takes 16 keys (a scale group) at a time and all query heads of a key/value head, on mma.sync m16n8k16 with fp16 operands, into which codes
// convert exactly:
//   S^T [16 keys x 8 heads] = K q        A: a lane holds 16-byte pieces of the keys g and g + 8. Which dimension an MMA's column k stands for is free, so
//                                        a lane's four consecutive codes are its four columns, and no shuffle or shared memory is needed
//   O^T [16 dims x 8 heads] += V^T P^T   A: a lane holds the same 8, 16 or 32 dimensions of the keys 2t, 2t + 1, 2t + 8, 2t + 9; bytes of two keys are
//                                        interleaved, which makes the operand's pairs. P^T comes from S^T by movmatrix
// so a lane's operands are pieces of the cache as they lie there. One TMA copy a group brings 16 tokens of a head (128 bytes of every kv_heads * 128 at heads of 128),
// three to six groups ahead of the warp that asked for them; group numbers and scales are looked up 32 at a time, one a lane. (32 rows of 8 heads behind 8,192 tokens,
// 537 MB: 104 us as int8, 98 as e4m3, 5.2 to 5.5 TB/s. With 16-byte copies by the lanes themselves it took 138 us, 133 without any arithmetic; with one group a warp under way in registers 135.)
// The next group's scores are issued beside one group's value products. int8 keys stay 1,152 too large, as they come out of their conversion: the
// scores' accumulators begin at -1,152 times the sum of the head's queries, so every term is exact and the fp32 sums are off by no more than the queries' own rounding.
// A group's key scale multiplies its scores, its value scale the weights: as fp16 they are 2^s * scale over the largest such product that the head has met, times 256: never above 2^15,
// and not small because of large values that the softmax passes over. The largest score, which sums of 2^(s - m) are relative to, is followed apart; both references
// move only when they have been passed by 7 (powers of two; sums are fp32). Queries are fp16 over a power of two of their own per head, so their size is no matter.
// 8 warps a CTA take groups in turn; a cluster of up to 16 CTAs splits a row's keys and merges through distributed shared memory, each CTA a
// share of the outputs. The group that the row's own token joins belongs to rank 0 alone, which settles its scales, rewrites it where they have grown and
// attends to it from shared memory; nobody else looks at it.
#include "cache8.cuh"
#include "tcgen05_util.cuh"

namespace {

constexpr int A1_SPLITS = 16, A1_WARPS = 8, A1_THREADS = 32 * A1_WARPS;
// groups that a warp has under way: as many as shared memory holds at two CTAs an SM (at one, where registers allow no more)
template <int KC, int NT> constexpr int kAhead = KC == 1 ? 6 : (KC == 2 && NT == 2) ? 6 : 3;
template <int KC, int VW> constexpr int kGroupBytes = 1024 * KC + 512 * VW;
constexpr float kWeightBits = 8.f, kFarScale = -60.f;

// 16 tokens of one head, `group` of the pool, from dimension d on
__device__ __forceinline__ void copy_tokens(uint32_t dst, const CUtensorMap* map, int d, int head, int group, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(d), "r"(head), "r"(0), "r"(group), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float cluster_load(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// KC: 16-code pieces of a key per lane (64 dimensions each). VW: words of a value per lane (32 dimensions each).
template <int KC> struct KeyCodes { uint32_t w[2][KC][4]; };                // keys g, g + 8
template <int VW> struct ValueCodes { uint32_t w[4][VW]; };                 // keys 2t, 2t + 1, 2t + 8, 2t + 9
// Where a lane's pieces lie in a group, from its first token's codes for the key/value head on.
struct Places { int k[2], v[4]; };
// `last`: the group's last token that may be read
__device__ __forceinline__ Places places_of(int kstride, int vstride, int piece, int last, int lane) {
    const int g = lane >> 2, t = lane & 3;
    Places p;
#pragma unroll
    for (int i = 0; i < 2; i++) p.k[i] = min(g + 8 * i, last) * kstride + 16 * t;
#pragma unroll
    for (int i = 0; i < 4; i++) p.v[i] = min(2 * t + (i & 1) + 8 * (i >> 1), last) * vstride + piece * g;
    return p;
}
// Where piece `chunk` (16 dimensions) of a group's token lies behind the group's copy: rows of 64 or 128 bytes with the copy's swizzle of that width, 128 dimensions
// after 128.
template <int SLABS> __device__ __forceinline__ int place_of(int token, int chunk) {
    if constexpr (SLABS == 1) return 64 * token + ((chunk ^ ((token >> 1) & 3)) << 4);
    else return (chunk >> 3) * (kScaleTokens * 128) + 128 * token + (((chunk ^ token) & 7) << 4);
}
template <int KC>
__device__ __forceinline__ void take_keys(KeyCodes<KC>& x, const uint8_t* from, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const uint4 u = *reinterpret_cast<const uint4*>(from + place_of<KC>(g + 8 * i, 4 * c + t));
            x.w[i][c][0] = u.x; x.w[i][c][1] = u.y; x.w[i][c][2] = u.z; x.w[i][c][3] = u.w;
        }
}
// `last`: what tokens behind it hold is taken as zero
template <int KC, int VW>
__device__ __forceinline__ void take_values(ValueCodes<VW>& x, const uint8_t* from, int last, int lane) {
    const int g = lane >> 2, t = lane & 3;
    from += 1024 * KC;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int token = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (VW == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(from + place_of<1>(token, g >> 1) + 8 * (g & 1));
            x.w[i][0] = u.x; x.w[i][1] = u.y;
        } else {
#pragma unroll
            for (int c = 0; c < VW / 4; c++) {
                const uint4 u = *reinterpret_cast<const uint4*>(from + place_of<2>(token, 8 * c + g));
                x.w[i][4 * c] = u.x; x.w[i][4 * c + 1] = u.y; x.w[i][4 * c + 2] = u.z; x.w[i][4 * c + 3] = u.w;
            }
        }
    }
    if (last < kScaleTokens - 1) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < VW; c++)
                if (2 * t + (i & 1) + 8 * (i >> 1) > last) x.w[i][c] = 0u;
    }
}
// The same from the row's own group, which lies in shared memory token by token.
template <int KC, int VW>
__device__ __forceinline__ void take_tail(KeyCodes<KC>& xk, ValueCodes<VW>& xv, const uint8_t* k, const uint8_t* v, const Places& p, int dk, int dv, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (64 * c + 16 * t < dk) u = *reinterpret_cast<const uint4*>(k + p.k[i] + 64 * c);
            xk.w[i][c][0] = u.x; xk.w[i][c][1] = u.y; xk.w[i][c][2] = u.z; xk.w[i][c][3] = u.w;
        }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (VW == 2) {
            uint2 u = make_uint2(0u, 0u);
            if (8 * g < dv) u = *reinterpret_cast<const uint2*>(v + p.v[i]);
            xv.w[i][0] = u.x; xv.w[i][1] = u.y;
        } else {
#pragma unroll
            for (int c = 0; c < VW / 4; c++) {
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (128 * c + 16 * g < dv) u = *reinterpret_cast<const uint4*>(v + p.v[i] + 128 * c);
                xv.w[i][4 * c] = u.x; xv.w[i][4 * c + 1] = u.y; xv.w[i][4 * c + 2] = u.z; xv.w[i][4 * c + 3] = u.w;
            }
        }
    }
}
// A word's codes as the keys' operand: int8 codes 1,152 too large, which the accumulators know.
template <bool I8> __device__ __forceinline__ void unpack_key(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (I8) {
        const uint32_t u = w ^ 0x80808080u;
        lo = __byte_perm(u, 0x64646464u, 0x4140);
        hi = __byte_perm(u, 0x64646464u, 0x4342);
    } else {
        unpack8<false>(w, lo, hi);
    }
}

// What a warp carries: per head 8 n + 2 t + e the references m (log2 of scores) and w (of scores times value scales), the sum l (this lane's keys), and O^T.
template <int VW, int NT>
struct State {
    float m[NT][2], w[NT][2], l[NT][2], o[NT][2 * VW][4];
};

// The products of a group's keys with the queries. from: what a head's accumulators begin with.
template <bool I8, int KC, int NT>
__device__ __forceinline__ void key_products(float (&s)[NT][4], const KeyCodes<KC>& x, const uint32_t (&q)[NT][KC][4][2], const float (&from)[NT][2]) {
#pragma unroll
    for (int n = 0; n < NT; n++) { s[n][0] = from[n][0]; s[n][1] = from[n][1]; s[n][2] = from[n][0]; s[n][3] = from[n][1]; }
#pragma unroll
    for (int c = 0; c < KC; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t a[4];
            unpack_key<I8>(x.w[0][c][j], a[0], a[2]);
            unpack_key<I8>(x.w[1][c][j], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; n++) mma_f16(s[n], a, q[n][c][j][0], q[n][c][j][1]);
        }
}
// Scores and weights of a group whose first key is `key0`, for the row at position p: b is P^T. qs: per head its queries' power of two; ks, vs: the group's scales.
template <int VW, int NT>
__device__ __forceinline__ void make_weights(State<VW, NT>& st, float (&s)[NT][4], uint32_t (&b)[NT][2], float ks, float vs, const float (&qs)[NT][2], const float (&slope)[NT][2], int key0, int p,
                                             int k_lo, int keep, int lane) {
    const int g = lane >> 2;
    const float back = (float)(p - key0 - g);
    const bool edge = key0 + kScaleTokens - 1 > p || (key0 < k_lo && key0 + kScaleTokens > keep);
    const float lv = (float)((int)(__float_as_uint(vs) >> 23) - 127);        // log2 of a power of two
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float f = qs[n][e] * ks;
            s[n][e] = fmaf(s[n][e], f, -slope[n][e] * back);
            s[n][2 + e] = fmaf(s[n][2 + e], f, -slope[n][e] * (back - 8.f));
        }
    if (edge) {
        const int k0 = key0 + g, k1 = k0 + 8;
        const bool out0 = k0 > p || (k0 < k_lo && k0 >= keep), out1 = k1 > p || (k1 < k_lo && k1 >= keep);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (out0) s[n][e] = -INFINITY;
                if (out1) s[n][2 + e] = -INFINITY;
            }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float mx = fmaxf(s[n][e], s[n][2 + e]);
            over |= mx > st.m[n][e] + 7.f || mx + lv > st.w[n][e] + 7.f;
        }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float mx = fmaxf(s[n][e], s[n][2 + e]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float nw = fmaxf(st.w[n][e], mx + lv), nm = fmaxf(st.m[n][e], mx), c = nm == -INFINITY ? 1.f : ex2(st.w[n][e] - nw);
                st.l[n][e] *= nm == -INFINITY ? 1.f : ex2(st.m[n][e] - nm);
                st.m[n][e] = nm;
                st.w[n][e] = nw;
#pragma unroll
                for (int i = 0; i < 2 * VW; i++) { st.o[n][i][e] *= c; st.o[n][i][2 + e] *= c; }
            }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float m = st.m[n][e] == -INFINITY ? 0.f : st.m[n][e], lift = st.m[n][e] == -INFINITY ? 0.f : st.w[n][e] - m;
            // (a group this far below the largest product weighs nothing; its part of l is made of the same exponentials)
            const float bits = fmaxf(lv - lift, kFarScale) + kWeightBits, u = bits - m;
            w[e] = ex2(s[n][e] + u);
            w[2 + e] = ex2(s[n][2 + e] + u);
            st.l[n][e] = fmaf(w[e] + w[2 + e], ex2(-bits), st.l[n][e]);
        }
        const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
        b[n][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
        b[n][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
    }
}
template <bool I8, int VW, int NT>
__device__ __forceinline__ void value_products(State<VW, NT>& st, const ValueCodes<VW>& x, const uint32_t (&b)[NT][2]) {
#pragma unroll
    for (int i = 0; i < VW; i++) {
        uint32_t a[4], c[4];                           // dimensions 4 i, 4 i + 1 of the lane's piece, then 4 i + 2, 4 i + 3
        unpack8<I8>(__byte_perm(x.w[0][i], x.w[1][i], 0x5140), a[0], a[1]);
        unpack8<I8>(__byte_perm(x.w[2][i], x.w[3][i], 0x5140), a[2], a[3]);
        unpack8<I8>(__byte_perm(x.w[0][i], x.w[1][i], 0x7362), c[0], c[1]);
        unpack8<I8>(__byte_perm(x.w[2][i], x.w[3][i], 0x7362), c[2], c[3]);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            mma_f16(st.o[n][2 * i], a, b[n][0], b[n][1]);
            mma_f16(st.o[n][2 * i + 1], c, b[n][0], b[n][1]);
        }
    }
}

// grid = (splits, kv_heads * passes, rows), clusters of `splits`. A pass is 8 NT query heads. append: the row's key and value enter the cache here
// (one pass then), otherwise they are in it.
template <bool I8, int KC, int VW, int NT>
__global__ void __launch_bounds__(A1_THREADS, KC == 4 || NT == 2 ? 1 : 2)
attention8_one_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const cmlb200_attn a, const float* __restrict__ qkv, int ld,
                      const int* __restrict__ row_pos, const int* __restrict__ row_slot, int append, __nv_bfloat16* __restrict__ out, int out_ld, int* status) {
    constexpr int HN = 8 * NT, AHEAD = kAhead<KC, NT>, GROUP = kGroupBytes<KC, VW>, DK = 64 * KC, DV = 32 * VW, PER = DK > DV ? DK / 32 : DV / 32;
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t* const groups_s = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    uint8_t* const ring = groups_s + (threadIdx.x >> 5) * (AHEAD * GROUP);   // the warp's groups under way
    uint8_t* const sm = groups_s + A1_WARPS * AHEAD * GROUP;
    const int dk = a.dim_ld, dv = a.vdim_ld;
    __half* q_s = reinterpret_cast<__half*>(sm);                             // [HN][DK]
    uint8_t* tail_k = sm + HN * DK * 2;                                      // [16][DK], [16][DV]: the row's own group
    uint8_t* tail_v = tail_k + kScaleTokens * DK;
    float* fresh = reinterpret_cast<float*>(tail_v + kScaleTokens * DV);     // [DK], [DV]: the row's own key and value
    float* w_acc = reinterpret_cast<float*>(groups_s);                       // [A1_WARPS][HN][DV] at the end, over all of the above
    __shared__ __align__(8) uint64_t full[A1_WARPS][AHEAD];
    __shared__ int abort_flag;
    __shared__ float w_m[A1_WARPS][HN], w_l[A1_WARPS][HN], c_m[HN], c_l[HN], q_unit[HN], q_sum[HN], tail_scale[2];
    __shared__ float2 red[A1_WARPS];
    if ((threadIdx.x & 31) == 0) {
        for (int j = 0; j < AHEAD; j++) mbar_init(smem_addr(&full[threadIdx.x >> 5][j]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) abort_flag = 0;
    __syncthreads();
    dep_trigger();
    dep_wait();
    const int splits = gridDim.x, rank = blockIdx.x, group = a.heads / a.kv_heads, passes = gridDim.y / a.kv_heads, kh = blockIdx.y / passes, pass = blockIdx.y % passes, r = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int h0 = kh * group + pass * HN, nh = min(HN, group - pass * HN);
    const float* row = qkv + (size_t)r * ld;
    const bool joins = append && rank == 0;
    // heads (queries, then on rank 0 the row's key and value) that a warp prepares: warp, warp + A1_WARPS, .. The first two's entries lane + 32 e are requested before
    // anything else is looked up
    auto request = [&](float (&y)[PER], int j) {
        const float* v = row;
        int n = 0;
        if (j < nh) { v = row + (h0 + j) * a.dim; n = a.dim; }
        else if (j == HN && joins) { v = row + (a.heads + kh) * a.dim; n = a.dim; }
        else if (j == HN + 1 && joins) { v = row + (a.heads + (a.keys_as_values ? 0 : a.kv_heads)) * a.dim + kh * a.vdim; n = a.vdim; }
#pragma unroll
        for (int e = 0; e < PER; e++) { const int d = lane + 32 * e; y[e] = d < n ? v[d] : 0.f; }
    };
    float now[PER], after[PER];
    request(now, warp);
    request(after, warp + A1_WARPS);
    const int p = row_pos[r], qw = a.heads * a.dim, kw = a.kv_heads * a.dim, shift = __ffs(a.block_size) - 1;
    const int* table = a.block_table + (size_t)row_slot[r] * a.table_ld;
    const int kstride = a.kv_heads * dk, vstride = a.kv_heads * dv;
    // the groups in sight, numbered from 0: those of the kept tokens, then those from k_lo on (one run where they meet)
    const int k_lo = first_key8(a, p), keep = a.keep, tail = p / kScaleTokens;
    int near = k_lo / kScaleTokens, kept = (min(keep, k_lo) + kScaleTokens - 1) / kScaleTokens;
    if (kept >= near) { near = 0; kept = 0; }
    const int groups = kept + tail - near + (append ? 0 : 1), step = splits * A1_WARPS;
    auto first_of = [&](int i) { return kScaleTokens * (i < kept ? i : near + i - kept); };
    KeyCodes<KC> xk;
    ValueCodes<VW> xv;
    constexpr int PIECE = VW == 2 ? 8 : 16;
    int i = rank * A1_WARPS + warp;
    // Where the warp's groups i, i + step, .. lie in the pools, 32 of them at a time, one a lane: the number of the group there, or -1; and their scales.
    const int i0 = i, per_page = a.block_size / kScaleTokens;
    auto look_up = [&](int n) {
        const int at = i0 + (n + lane) * step;
        if (at >= groups) return -1;
        const int first = first_of(at);
        return table[first >> shift] * per_page + (first & (a.block_size - 1)) / kScaleTokens;
    };
    auto scale_of = [&](const float* scales, int where) { return where < 0 ? 0.f : scales[(size_t)where * a.kv_heads + kh]; };
    int lie = look_up(0), lie_next = -1;
    const int own_page = table[p >> shift];
    // the warp's group number n into place `at` of the ring
    auto fetch = [&](int n, bool further, int at) {
        const int where = __shfl_sync(0xffffffffu, further ? lie_next : lie, n & 31);
        if (where >= 0 && lane == 0) {
            const uint32_t to = smem_addr(ring) + at * GROUP, bar = smem_addr(&full[warp][at]);
            mbar_expect_tx(bar, GROUP);
#pragma unroll
            for (int c = 0; c < (KC + 1) / 2; c++) copy_tokens(to + 2048 * c, &kmap, 128 * c, kh, where, bar);
#pragma unroll
            for (int c = 0; c < (VW + 3) / 4; c++) copy_tokens(to + 1024 * KC + 2048 * c, &vmap, 128 * c, kh, where, bar);
        }
    };
#pragma unroll
    for (int at = 0; at < AHEAD; at++) fetch(at, false, at);       // under way while the queries are made
    float ks = scale_of(a.k_scale, lie), vs = scale_of(a.v_scale, lie), ks_next = 0.f, vs_next = 0.f;

    // ---- the row's queries, and on rank 0 its key and value
    const size_t own = ((size_t)own_page << shift) + (p & (a.block_size - 1)), own_group = own / kScaleTokens * a.kv_heads + kh;
    const int off = p & (kScaleTokens - 1);
    uint8_t* kd = static_cast<uint8_t*>(a.k_pool) + ((own - off) * a.kv_heads + kh) * dk;
    uint8_t* vd = static_cast<uint8_t*>(a.v_pool) + ((own - off) * a.kv_heads + kh) * dv;
    constexpr int OLD = (kScaleTokens * (DK + DV) / 16 + A1_THREADS - 1) / A1_THREADS;
    uint4 old[OLD];                                    // piece threadIdx.x + A1_THREADS j of the group: token i / pieces, piece i % pieces
    const int kc = dk >> 4, pieces = kc + (dv >> 4);
    float was_k = 0.f, was_v = 0.f;
    if (joins && off) {
        was_k = a.k_scale[own_group];
        was_v = a.v_scale[own_group];
#pragma unroll
        for (int j = 0; j < OLD; j++) {
            const int e = threadIdx.x + A1_THREADS * j, tok = e / pieces, c = e - tok * pieces;
            if (tok < off) old[j] = *reinterpret_cast<const uint4*>(c < kc ? kd + (size_t)tok * kstride + 16 * c : vd + (size_t)tok * vstride + 16 * (c - kc));
        }
    }
    float iq = 1.0f, ik = 1.0f;
    if (!a.head_norm && (a.q_norm || a.k_norm)) {
        const float2 ss = block_sum2(a.q_norm ? square_share(row, qw) : 0.f, a.k_norm && joins ? square_share(row + qw, kw) : 0.f, red);
        if (a.q_norm) iq = 1.0f / sqrtf(ss.x / (float)qw + a.eps);
        if (a.k_norm) ik = 1.0f / sqrtf(ss.y / (float)kw + a.eps);
    }
    const float temp = a.temp_every > 0.f ? 1.0f + a.temp_coef * logf(floorf((float)(p + 1) / a.temp_every) + 1.0f) : 1.0f;
    // what a warp does with one head: entries lane + 32 j, normed and turned
    auto prepare = [&](float (&y)[PER], int n, const float* norm, float inv, bool head_norm, bool turns) {
        if (head_norm) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < PER; j++) ss = fmaf(y[j], y[j], ss);
            inv = 1.0f / sqrtf(lane_sum(ss) / (float)n + a.eps);
        }
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int d = lane + 32 * j;
            y[j] *= inv * (norm && d < n ? norm[d] : 1.0f);
            if (turns) {
                const float z = __shfl_xor_sync(0xffffffffu, y[j], 1);
                if (d < a.rot_dims) {
                    float c, s;
                    sincosf((float)p * a.freq[d >> 1], &s, &c);
                    y[j] = (d & 1) ? y[j] * c + z * s : y[j] * c - z * s;
                }
            }
        }
    };
    for (int j = warp; j < HN + (joins ? 2 : 0); j += A1_WARPS) {
        float y[PER], most = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) { y[e] = now[e]; now[e] = after[e]; }
        if (HN > A1_WARPS) request(after, j + 2 * A1_WARPS);
        if (j < HN) {
            if (j < nh) {
                prepare(y, a.dim, a.q_norm ? a.q_norm + (a.head_norm ? 0 : (h0 + j) * a.dim) : nullptr, iq, a.q_norm && a.head_norm, a.freq != nullptr);
            }
#pragma unroll
            for (int e = 0; e < PER; e++) { y[e] *= temp * a.scale * kLog2e; most = fmaxf(most, fabsf(y[e])); }
            most = lane_max(most);
            // a power of two that leaves 1 <= largest < 2 (2^-126 at least, so that its inverse is finite)
            const float unit = most > 0.f ? __uint_as_float(max(min(__float_as_uint(most) & 0x7F800000u, 0x7E000000u), 0x00800000u)) : 1.0f, inv = 1.0f / unit;
            float sum = 0.f;                           // of the queries as they are rounded
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const __half z = __float2half_rn(y[e] * inv);
                if (lane + 32 * e < DK) q_s[j * DK + lane + 32 * e] = z;
                sum += __half2float(z);
            }
            sum = lane_sum(sum);
            if (lane == 0) { q_unit[j] = unit; q_sum[j] = sum; }
        } else {
            const bool key = j == HN;
            if (key) prepare(y, a.dim, a.k_norm ? a.k_norm + (a.head_norm ? 0 : kh * a.dim) : nullptr, ik, a.k_norm && a.head_norm, a.freq != nullptr);
            else prepare(y, a.vdim, nullptr, 1.0f, false, false);
#pragma unroll
            for (int e = 0; e < PER; e++) { y[e] = cached8(y[e]); most = fmaxf(most, fabsf(y[e])); }
            most = lane_max(most);
            if (lane == 0) tail_scale[key ? 0 : 1] = scale8_for<I8>(most);
#pragma unroll
            for (int e = 0; e < PER; e++) if (lane + 32 * e < (key ? DK : DV)) fresh[(key ? 0 : DK) + lane + 32 * e] = y[e];
        }
    }
    __syncthreads();
    if (joins) {
        const float sk = fmaxf(tail_scale[0], was_k), sv = fmaxf(tail_scale[1], was_v), rk = off ? was_k / sk : 1.f, rv = off ? was_v / sv : 1.f, ik8 = 1.0f / sk, iv8 = 1.0f / sv;
#pragma unroll
        for (int j = 0; j < OLD; j++) {
            const int e = threadIdx.x + A1_THREADS * j, tok = e / pieces, c = e - tok * pieces;
            if (tok >= kScaleTokens) break;
            const bool key = c < kc;
            const float ratio = key ? rk : rv;
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (tok < off) {
                u = old[j];
                if (ratio != 1.f) { u.x = rescale8<I8>(u.x, ratio); u.y = rescale8<I8>(u.y, ratio); u.z = rescale8<I8>(u.z, ratio); u.w = rescale8<I8>(u.w, ratio); }
            } else if (tok == off) {
                const float* f = key ? fresh + 16 * c : fresh + DK + 16 * (c - kc);
                const float inv = key ? ik8 : iv8;
                u.x = pack8<I8>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
                u.y = pack8<I8>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
                u.z = pack8<I8>(f[8] * inv, f[9] * inv, f[10] * inv, f[11] * inv);
                u.w = pack8<I8>(f[12] * inv, f[13] * inv, f[14] * inv, f[15] * inv);
            }
            *reinterpret_cast<uint4*>(key ? tail_k + tok * DK + 16 * c : tail_v + tok * DV + 16 * (c - kc)) = u;
            if (tok == off || (tok < off && ratio != 1.f)) *reinterpret_cast<uint4*>(key ? kd + (size_t)tok * kstride + 16 * c : vd + (size_t)tok * vstride + 16 * (c - kc)) = u;
        }
        __syncthreads();                               // (all have read tail_scale)
        if (threadIdx.x == 0) { a.k_scale[own_group] = sk; a.v_scale[own_group] = sv; tail_scale[0] = sk; tail_scale[1] = sv; }
        __syncthreads();
    }
    uint32_t q[NT][KC][4][2];
    float qs[NT][2], slope[NT][2], from_[NT][2];
    State<VW, NT> st;
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint2 u = *reinterpret_cast<const uint2*>(q_s + (8 * n + g) * DK + 64 * c + 16 * t + 4 * j);
                q[n][c][j][0] = u.x;
                q[n][c][j][1] = u.y;
            }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int j = 8 * n + 2 * t + e;
            qs[n][e] = q_unit[j];
            from_[n][e] = I8 ? -1152.f * q_sum[j] : 0.f;
            slope[n][e] = a.slopes && j < nh ? a.slopes[h0 + j] * kLog2e : 0.f;
            st.m[n][e] = -INFINITY;
            st.w[n][e] = -INFINITY;
            st.l[n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * VW; k++) { st.o[n][k][e] = 0.f; st.o[n][k][2 + e] = 0.f; }
        }
    }
    // ---- the cached groups
    float sc[NT][4];
    uint32_t pb[NT][2];
    // The next group's scores are made beside the values' products of one: two chains of MMAs that do not wait for each other. (Behind the last group there are
    // scores of whatever lies in the ring; nobody looks at them.)
    uint32_t phase = 0;
    bool ok = true;
    auto scores = [&](int at, bool there) {
        if (there) ok = __all_sync(0xffffffffu, mbar_wait(smem_addr(&full[warp][at]), phase, &abort_flag, 9, status));
        if (!ok) return;
        take_keys<KC>(xk, ring + at * GROUP, lane);
        key_products<I8, KC, NT>(sc, xk, q, from_);
    };
    scores(0, i < groups);
    int at = 0;
    for (int n = 0; i < groups && ok; i += step, n++) {
        make_weights<VW, NT>(st, sc, pb, __shfl_sync(0xffffffffu, ks, n & 31), __shfl_sync(0xffffffffu, vs, n & 31), qs, slope, first_of(i), p, k_lo, keep, lane);
        take_values<KC, VW>(xv, ring + at * GROUP, append ? kScaleTokens - 1 : p - first_of(i), lane);
        __syncwarp();                                  // (all lanes have what they need of the place)
        fetch(n + AHEAD, (n & 31) >= 32 - AHEAD, at);
        if (++at == AHEAD) { at = 0; phase ^= 1; }
        // the next 32 groups' places, then their scales, long before they are needed
        if ((n & 31) == 8) lie_next = look_up((n & ~31) + 32);
        if ((n & 31) == 16) { ks_next = scale_of(a.k_scale, lie_next); vs_next = scale_of(a.v_scale, lie_next); }
        if ((n & 31) == 31) { lie = lie_next; ks = ks_next; vs = vs_next; }
        scores(at, i + step < groups);
        value_products<I8, VW, NT>(st, xv, pb);
    }
    if (joins && warp == 0) {
        take_tail<KC, VW>(xk, xv, tail_k, tail_v, places_of(DK, DV, PIECE, off, lane), dk, dv, lane);
        key_products<I8, KC, NT>(sc, xk, q, from_);
        make_weights<VW, NT>(st, sc, pb, tail_scale[0], tail_scale[1], qs, slope, tail * kScaleTokens, p, k_lo, keep, lane);
        value_products<I8, VW, NT>(st, xv, pb);
    }
    if (!ok) {                                         // a wait gave up, and has said so: what is under way gets as long again
        for (int k = 0; k < AHEAD && i + k * step < groups; k++) {
            for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(smem_addr(&full[warp][at]), phase); it++) {}
            if (++at == AHEAD) { at = 0; phase ^= 1; }
        }
    }
    // ---- merge the warps, then the CTAs of the cluster
    __syncthreads();                                   // queries and tail are done with
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float l = st.l[n][e];
            const float unit = st.m[n][e] == -INFINITY ? 0.f : ex2(st.w[n][e] - st.m[n][e] - kWeightBits);
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int j = 8 * n + 2 * t + e;
            if (g == 0) { w_m[warp][j] = st.m[n][e]; w_l[warp][j] = l; }
            float* d = w_acc + (warp * HN + j) * DV;
#pragma unroll
            for (int w = 0; w < VW; w++) {
                const int at = VW == 2 ? 8 * g + 4 * w : 128 * (w / 4) + 16 * g + 4 * (w % 4);
                *reinterpret_cast<float4*>(d + at) = make_float4(st.o[n][2 * w][e] * unit, st.o[n][2 * w][2 + e] * unit, st.o[n][2 * w + 1][e] * unit, st.o[n][2 * w + 1][2 + e] * unit);
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * DV; e += A1_THREADS) {
        const int j = e / DV;
        float mx = w_m[0][j];
#pragma unroll
        for (int w = 1; w < A1_WARPS; w++) mx = fmaxf(mx, w_m[w][j]);
        float v = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < A1_WARPS; w++) {
            const float mw = w_m[w][j], c = mw == -INFINITY ? 0.f : exp2f(mw - mx);
            v = fmaf(w_acc[w * HN * DV + e], c, v);
            sum = fmaf(w_l[w][j], c, sum);
        }
        w_acc[e] = v;                                  // element e of warp 0's part is read and written by this thread alone
        if (e - j * DV == 0) { c_m[j] = mx; c_l[j] = sum; }
    }
    if (splits > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    for (int e = rank * A1_THREADS + threadIdx.x; e < nh * DV; e += splits * A1_THREADS) {
        const int j = e / DV, d = e - j * DV;
        float v, sum, mx;
        if (splits > 1) {
            mx = -INFINITY; v = 0.f; sum = 0.f;
            for (int s0 = 0; s0 < splits; s0 += 8) {
                float ms[8], ls[8], vs[8];
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    ms[s] = -INFINITY; ls[s] = 0.f; vs[s] = 0.f;
                    if (s0 + s < splits) {
                        ms[s] = cluster_load(cluster_addr(c_m + j, s0 + s));
                        ls[s] = cluster_load(cluster_addr(c_l + j, s0 + s));
                        vs[s] = cluster_load(cluster_addr(w_acc + e, s0 + s));
                    }
                }
                float top = mx;
#pragma unroll
                for (int s = 0; s < 8; s++) top = fmaxf(top, ms[s]);
                const float was = mx == -INFINITY ? 0.f : exp2f(mx - top);
                v *= was;
                sum *= was;
                mx = top;
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    const float c = ms[s] == -INFINITY ? 0.f : exp2f(ms[s] - mx);
                    v = fmaf(vs[s], c, v);
                    sum = fmaf(ls[s], c, sum);
                }
            }
        } else {
            v = w_acc[e]; sum = c_l[j]; mx = c_m[j];
        }
        if (a.sink) {                                  // it carries no value
            const float sk = (a.sinks ? a.sinks[h0 + j] : 0.f) * kLog2e, mt = fmaxf(mx, sk), c = exp2f(mx - mt);
            v *= c;
            sum = sum * c + exp2f(sk - mt);
        }
        v = v / sum * (a.out_scale == 0.f ? 1.f : a.out_scale);
        if (a.gate_col >= 0) v *= sigmoidf(row[a.gate_col + h0 + j]);
        if (d < a.vdim) out[(size_t)r * out_ld + (h0 + j) * a.vdim + d] = __float2bfloat16_rn(v);
    }
    if (splits > 1) {                                  // nobody leaves while others read its shared memory
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// A pool as [groups of 16 tokens][token][head][dimension], its end open: group numbers come from block tables. Rows of up to `width` codes, zeros behind dim_ld.
int map_pool(CUtensorMap* map, const void* pool, int kv_heads, int dim_ld, int width) {
    const int row = width < 128 ? width : 128;
    const cuuint64_t head = (cuuint64_t)dim_ld, token = head * kv_heads, dims[4] = {head, (cuuint64_t)kv_heads, kScaleTokens, 1ull << 31}, strides[3] = {head, token, token * kScaleTokens};
    const cuuint32_t box[4] = {(cuuint32_t)row, 1, kScaleTokens, 1}, one[4] = {1, 1, 1, 1};
    EncodeTiledFn encode;
    const int rc = get_encoder(&encode);
    if (rc) return rc;
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(pool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CMLB_REQUIRE(r == CUDA_SUCCESS, "cmlb200_attention_one: cuTensorMapEncodeTiled failed with %d for %d heads of %d", (int)r, kv_heads, dim_ld);
    return CMLB200_OK;
}

template <bool I8, int KC, int VW, int NT>
int launch_one(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int rows, int keys, int passes, int append, __nv_bfloat16* d_out, int out_ld,
               cudaStream_t st) {
    constexpr size_t HN = 8 * NT, DK = 64 * KC, DV = 32 * VW;
    constexpr size_t before = HN * DK * 2 + kScaleTokens * (DK + DV) + 4 * (DK + DV) + A1_WARPS * kAhead<KC, NT> * kGroupBytes<KC, VW>, after = 4 * A1_WARPS * HN * DV, smem = 1024 + (before > after ? before : after);
    static size_t attr[kMaxDevices] = {};
    auto kern = attention8_one_kernel<I8, KC, VW, NT>;
    CMLB_CUDA(cmlb_ensure_smem(kern, smem, attr));
    // How many CTAs share a row's keys: what takes least by an estimate in units of a warp's time for a group (1.2 us where few are under way): 6 for a CTA's
    // beginning and end, times the waves, where clusters of a size share the device with as many as fit its groups of SMs. (One row of 8 heads behind 32,000
    // tokens: 45 us by 8, 35 by 16. 8 behind 2,000: 15.9 us; when a group took a third longer, 18.3 by 4, 24.4 by 2, 27.7 by 8, which takes two waves.)
    static int room[kMaxDevices][A1_SPLITS + 1] = {};
    if (!room[cmlb_device_index()][1]) CMLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    const long long base = (long long)rows * a->kv_heads * passes, groups = (keys + kScaleTokens - 1) / kScaleTokens;
    long long best = 0;
    int splits = 1;
    for (int k = 1; k <= A1_SPLITS && (k == 1 || groups > (k - 1) * A1_WARPS); k++) {
        int* fit = &room[cmlb_device_index()][k];
        if (!*fit) *fit = cluster_room((const void*)kern, k, A1_THREADS, smem);
        if (*fit < 0) continue;
        const long long t = (base + *fit - 1) / *fit * (6 + (groups + k * A1_WARPS - 1) / (k * A1_WARPS));
        if (k == 1 || t < best) { best = t; splits = k; }
    }
    CUtensorMap kmap, vmap;
    int* status;
    int rc = map_pool(&kmap, a->k_pool, a->kv_heads, a->dim_ld, DK);
    if (!rc) rc = map_pool(&vmap, a->v_pool, a->kv_heads, a->vdim_ld, DV);
    if (!rc) rc = cmlb_attention8_status_word(&status);
    if (rc) return rc;
    CMLB_CUDA(launch_chain(kern, dim3(splits, a->kv_heads * passes, rows), dim3(A1_THREADS), smem, splits, st, kmap, vmap, *a, d_qkv, ld, d_row_pos, d_row_slot, append, d_out, out_ld, status));
    return CMLB200_OK;
}

}  // namespace

int cmlb_attention8_one(const cmlb200_attn* a, const float* d_qkv, int ld, const int* d_row_pos, const int* d_row_slot, int rows, int max_keys, __nv_bfloat16* d_out, int out_ld,
                        cudaStream_t st) {
    const int widest = a->dim_ld > a->vdim_ld ? a->dim_ld : a->vdim_ld;
    // (heads of 256 with 16 of them in a pass would not fit registers: their keys are read twice)
    const int group = a->heads / a->kv_heads, nt = group <= 8 || widest > 128 ? 1 : 2, passes = (group + 8 * nt - 1) / (8 * nt), append = passes == 1;
    CMLB_REQUIRE((long long)a->kv_heads * passes <= 65535, "cmlb200_attention_one: too many heads");
    if (!append) {                                     // several passes read the row's own group: it is written by a launch of its own
        const int rc = cmlb_cache8_append(a, const_cast<float*>(d_qkv), ld, d_row_pos, d_row_slot, 0, rows, true, false, st);
        if (rc) return rc;
    }
    const int reach = a->chunk > 0 ? a->chunk : a->window;
    const int keys = (reach > 0 && reach < max_keys - a->keep) ? reach + a->keep : max_keys;
#define A1_ARGS a, d_qkv, ld, d_row_pos, d_row_slot, rows, keys, passes, append, d_out, out_ld, st
#define A1_HEADS(I8, KC, VW) return nt == 1 ? launch_one<I8, KC, VW, 1>(A1_ARGS) : launch_one<I8, KC, VW, 2>(A1_ARGS)
#define A1_SIZES(I8)                            \
    do {                                         \
        if (widest <= 64) A1_HEADS(I8, 1, 2);    \
        if (widest <= 128) A1_HEADS(I8, 2, 4);   \
        return launch_one<I8, 4, 8, 1>(A1_ARGS); \
    } while (0)
    if (a->cache_dtype == CMLB200_DT_I8) A1_SIZES(true);
    A1_SIZES(false);
#undef A1_SIZES
#undef A1_HEADS
#undef A1_ARGS
}
