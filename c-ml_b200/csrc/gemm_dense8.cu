// Prompt-sized products of int8 weights and int8 rows on the 5th-generation tensor cores: whole numbers in 32 bits in tensor memory, then
// y = sum * (sx[m] sw[n]) (+ bias, cap), or bf16 act(gate) * up.
//
// Weight rows are the MMA's "M" side (operand A), rows of x its "N" side: a lane of tensor memory is a channel, a column a token. A channel's scale and bias are then a lane's own
// registers, 32 lanes store 32 neighbouring outputs of a token with nothing transposed, a gate row and its up row are 16 lanes apart, and the number of tokens of a
// tile is any multiple of 16 up to 256.
//   warp 0      one lane issues TMA loads of both operands (256 columns a stage, as two blocks of 128 with 128-byte swizzle that one load brings) into a ring of stages that runs
//               on across tiles; weights of the first stages before the launch in front has ended
//   warp 1      owns tensor memory; an elected lane issues tcgen05.mma kind::i8 (128 or 256 x NX x 32)
//   warps 2-9   epilogue, two a quarter of tensor memory's lanes
// Three forms (pick_shape):
//   pairs       256 channels by up to 256 tokens, a pair of CTAs (cta_group::2): each has 128 channels and half of the tokens' codes. Persistent, two accumulators in turn.
//   single      128 channels, persistent, the same.
//   split       where tiles are fewer than SMs a cluster of 2 to 8 CTAs shares the columns of a tile. Each finishes its share of the tokens: the others store their sums of those
//               into its shared memory. Since they are whole numbers the order of adding makes no difference.
// What bounds it. Many tokens: an SM reads 64 KB from L2 for the 1,024 cycles of MMAs of a stage of 256 x 256 x 256, and gets them in about 1,250 (13.5 TB/s in all): tensor cores 85 % busy, 4,096 tokens of
// 8192x8192 175 us; for seconds on end the power limit, 4,096 of 8192x28672 640 us and 3.0 POP/s. Few tokens: the weight's bytes, and beside them the codes' launch, 0.7 us from its end to the first
// MMA, 0.4 us behind the last, 0.6 to 2.5 us of epilogue (77 of 11008x4096 13.7 us, the bytes 7.3; 500 of 6144x4096 18.1; 256 of 4096x4096 11.5).
// The one thread that loads and the warp that issues MMAs were what took the time before: places found by division 900 cycles a block, a wait, a fence and a commit for every 128 columns 500.
// No load is multicast. Every wait on an mbarrier is bounded; on expiry the CTA raises a status word (cmlb200_dense8_status), waits for its copies and MMAs in flight, frees its tensor
// memory and returns.
#include <math.h>

#include "dense8.cuh"
#include "status_word.cuh"
#include "tcgen05_util.cuh"

namespace {

constexpr int BK8 = 128, BLOCKS = 2, CH = 128;         // columns of a block, blocks of a stage, channels of a CTA
constexpr int EPI = 8, THREADS8 = 64 + EPI * 32;
constexpr int A8 = CH * BK8, MOST_STAGES = 8, ROOM8 = 220 * 1024;
constexpr int SCALES8 = 1024, HEAD8 = SCALES8 + EPI * 512;                    // in front of the stages: barriers and words, then the epilogue warps' scales of tokens

__device__ __forceinline__ bool wait8(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, int* status) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, code, status));
}
// for what is under way whoever has given up
__device__ __forceinline__ void drain8(uint32_t bar, uint32_t parity) {
    for (uint32_t it = 0; it < SPIN_LIMIT && !mbar_try(bar, parity); ++it)
        if (it > 1024) __nanosleep(32);
}
template <bool PAIR>
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    if (PAIR)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                     ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                     ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void commit8(uint32_t bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        umma_commit(bar);
}
// eight columns of a warp's lanes; there when tmem_there() has returned
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, int (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_there(int (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) : : "memory");
}
// `BLOCKS` blocks of 128 columns of a box of rows
__device__ __forceinline__ void load_blocks(uint32_t dst, const CUtensorMap* map, int row, int block, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(block), "r"(bar) : "memory");
}
// Arrives at the same barrier of the pair's first CTA. What the arrival stands for lies in this SM's own memory, which its half of the MMA reads: no release for the cluster.
__device__ __forceinline__ void arrive_first(uint32_t bar) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(bar));
    asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory");
}
__device__ __forceinline__ void whole_cluster() { asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

struct Gemm8 {
    Out8 out;
    int M, N, loads, NX, tiles_m, tiles, stages, glu;
    int* status;
};

// Tile number -> token tile, channel tile: groups of 8 token tiles share a sweep over the channels, so that the CTAs working at one time read few distinct slabs.
__device__ __forceinline__ void tile8(int i, int tiles_m, int tiles, int& tm, int& tn) {
    const int cols = tiles / tiles_m, per = 8 * cols, gq = i / per, in = i - gq * per, rows = min(8, tiles_m - gq * 8);
    tm = gq * 8 + in % rows;
    tn = in / rows;
}

template <bool PAIR>
__global__ void __launch_bounds__(THREADS8, 1)
gemm_dense8_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const Gemm8 p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t bars = smem_u32(smem), sbase = bars + HEAD8;
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (MOST_STAGES + s); };
    auto acc_full = [&](int b) { return bars + 8 * (2 * MOST_STAGES + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (2 * MOST_STAGES + 2 + b); };
    const uint32_t drained = bars + 8 * (2 * MOST_STAGES + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 8 * (2 * MOST_STAGES + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int second = PAIR ? (int)rank : 0, first_tile = blockIdx.x / ranks, step = gridDim.x / ranks;
    if (PAIR) { rank = 0; ranks = 1; }
    const int kb0 = (int)((long)p.loads * rank / ranks), nkb = (int)((long)p.loads * (rank + 1) / ranks) - kb0;
    const int my_tiles = first_tile < p.tiles ? (p.tiles - first_tile + step - 1) / step : 0, total = my_tiles * nkb;
    const int b_rows = PAIR ? p.NX / 2 : p.NX, blocks_a = BLOCKS * A8, stage = blocks_a + BLOCKS * b_rows * BK8, S = p.stages;
    const int acc = p.NX <= 32 ? 32 : p.NX <= 64 ? 64 : p.NX <= 128 ? 128 : 256;

    // places of the next stages to load, counted: with divisions the one thread took 900 cycles a stage
    struct Place { int tile, k, row; } w = {first_tile, 0, 0}, x = {first_tile, 0, 0};
    auto tile_row = [&](int tile, bool of_tokens) {
        int tm, tn;
        tile8(tile, p.tiles_m, p.tiles, tm, tn);
        return of_tokens ? tm * p.NX + second * b_rows : (PAIR ? 2 * CH : CH) * tn + CH * second;
    };
    auto next = [&](Place& at, bool of_tokens) {
        if (++at.k == nkb) {
            at.k = 0;
            at.tile += step;
            if (at.tile < p.tiles) at.row = tile_row(at.tile, of_tokens);
        }
    };
    auto weights = [&](uint32_t to, uint32_t bar) {
        mbar_expect_tx(bar, (uint32_t)stage);
        load_blocks(to, &wmap, w.row, (kb0 + w.k) * BLOCKS, bar);
        next(w, false);
    };
    auto tokens = [&](uint32_t to, uint32_t bar) {
        load_blocks(to + blocks_a, &xmap, x.row, (kb0 + x.k) * BLOCKS, bar);
        next(x, true);
    };
    const int ahead = min(S, total);
    if (threadIdx.x == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&xmap) : "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) { mbar_init(full(s), PAIR && !second ? 2 : 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), PAIR ? 2 * EPI : EPI); }
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        w.row = tile_row(first_tile, false);
        x.row = tile_row(first_tile, true);
        for (int it = 0; it < ahead; it++) weights(sbase + it * stage, full(it));
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * acc)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * acc)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    dep_trigger();
    tmem_fence_before();
    __syncthreads();
    if (PAIR) whole_cluster();                         // its barriers and columns, too
    tmem_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            dep_wait();
            asm volatile("fence.proxy.async.global;" ::: "memory");
            for (int it = 0; it < ahead; it++) tokens(sbase + it * stage, full(it));
            int it = ahead, s = 0;
            uint32_t phase = 0, to = sbase;
            for (; it < total; it++) {
                if (!mbar_wait(empty(s), phase, abort_flag, 1, p.status)) break;
                weights(to, full(s));
                tokens(to, full(s));
                to += stage;
                if (++s == S) { s = 0; phase ^= 1; to = sbase; }
            }
            // no copy outlives its CTA (a pair's first CTA: its barriers also wait for the second one's arrivals, which come or are given up)
            for (int i = max(0, it - S); i < it; i++) drain8(full(i % S), (i / S) & 1);
        }
    } else if (warp == 1) {
        // kind::i8: D s32, A and B signed
        const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.NX >> 3) << 17) | ((uint32_t)((PAIR ? 2 * CH : CH) >> 4) << 24);
        const uint64_t desc0 = make_desc(sbase);
        const uint32_t b_block = (uint32_t)(b_rows * BK8) >> 4;
        int s = 0, done = 0;
        uint32_t phase = 0;
        bool ok = true;
        if (PAIR && second) {                          // tells the first CTA what has come to this one
            for (int it = 0; it < total && ok; it++) {
                ok = wait8(full(s), phase, abort_flag, 2, p.status);
                if (ok && lane == 0) arrive_first(full(s));
                __syncwarp();
                if (++s == S) { s = 0; phase ^= 1; }
            }
        } else {
            for (; done < my_tiles && ok; done++) {
                const int b = done & 1;
                ok = wait8(acc_empty(b), ((done >> 1) & 1) ^ 1, abort_flag, 3, p.status);
                if (!ok) break;
                tmem_fence_after();
                for (int k = 0; k < nkb; k++) {
                    ok = wait8(full(s), phase, abort_flag, 4, p.status);
                    if (!ok) break;
                    tmem_fence_after();
                    const uint64_t ad = desc0 + (uint64_t)(uint32_t)(s * (stage >> 4)), bd = ad + (uint64_t)(blocks_a >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BLOCKS * BK8 / 32; kk++)
                            umma_i8<PAIR>(tmem_base + (uint32_t)(b * acc), ad + (uint64_t)((kk >> 2) * (A8 >> 4) + 2 * (kk & 3)), bd + (uint64_t)((kk >> 2) * b_block + 2 * (kk & 3)), idesc,
                                          (k | kk) ? 1u : 0u);
                        commit8<PAIR>(empty(s));
                    }
                    __syncwarp();
                    if (++s == S) { s = 0; phase ^= 1; }
                }
                if (elect_one()) commit8<PAIR>(acc_full(b));
                __syncwarp();
            }
            if (elect_one()) commit8<PAIR>(drained);   // tensor memory and the stages outlive the MMAs
            __syncwarp();
            drain8(drained, 0);
        }
    } else {
        dep_wait();
        const int q = warp & 3, half = (warp - 2) >> 2, ch = q * 32 + lane, up = lane >> 4;
        const uint32_t lanes = tmem_base + ((uint32_t)(q * 32) << 16);
        // a cluster: rank d finishes tokens d * share .. of the tile; the other ranks' sums of them come to [rank in front of it or behind][share / 4][128][4] where its stages were
        const int share = (p.NX + 8 * (int)ranks - 1) / (8 * (int)ranks) * 8;
        int* const sums = reinterpret_cast<int*>(smem + HEAD8);
        float* const sxs = reinterpret_cast<float*>(smem + SCALES8) + (warp - 2) * 128;        // of this warp's tokens, in the order it comes to them
        for (int done = 0; done < my_tiles; done++) {
            const int b = done & 1;
            int tm, tn;
            tile8(first_tile + done * step, p.tiles_m, p.tiles, tm, tn);
            const int n = tn * (PAIR ? 2 * CH : CH) + CH * second + ch, m0 = tm * p.NX, most = min(p.NX, p.M - m0);
            const float sw = n < p.N ? p.out.wscale[n] : 0.f, bias = p.out.bias && n < p.N ? p.out.bias[n] : 0.f;
            const int c_lo = (int)rank * share, c_hi = min(most, ranks > 1 ? c_lo + share : p.NX);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = c_lo + half * 8 + (4 * i + (lane >> 3)) * 16 + (lane & 7);
                sxs[i * 32 + lane] = c < c_hi ? p.out.xscale[m0 + c] : 0.f;
            }
            __syncwarp();
            const bool there = wait8(acc_full(b), (done >> 1) & 1, abort_flag, 5, p.status);
            tmem_fence_after();
            const uint32_t acc_at = lanes + (uint32_t)(b * acc);
            if (ranks > 1) {
                __syncwarp();
                whole_cluster();                       // everyone's MMAs are through with the stages
                if (there)
#pragma unroll 1
                    for (int d = 1; d < (int)ranks; d++) {
                        const int to = ((int)rank + d) & ((int)ranks - 1), slot = (int)rank < to ? (int)rank : (int)rank - 1, end = min(share, p.NX - to * share);
                        const uint32_t base = cluster_addr(sums + (size_t)(slot * share) * CH + ch * 4, to);
                        int v[8], c = half * 8;
                        if (c < end) tmem_ld8(acc_at + (uint32_t)(to * share + c), v);
#pragma unroll 1
                        for (; c < end; c += 16) {
                            int u[8];
                            tmem_there(v);
#pragma unroll
                            for (int j = 0; j < 8; j++) u[j] = v[j];
                            if (c + 16 < end) tmem_ld8(acc_at + (uint32_t)(to * share + c + 16), v);
#pragma unroll
                            for (int j = 0; j < 8; j += 4)
                                asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(base + (uint32_t)((c + j) * CH * 4)), "r"(u[j]), "r"(u[j + 1]), "r"(u[j + 2]), "r"(u[j + 3]) : "memory");
                        }
                    }
                __syncwarp();
                whole_cluster();                       // what the others have is here
            }
            if (!there) break;
            // Eight tokens a turn in a small loop: nothing of a kernel's code is cached when it begins, and this is where most of it would be (unrolled over 32 tokens: 4 to 5 us for 128)
            const int col = (n >> 5) * 16 + (lane & 15);
            const float4* sx4 = reinterpret_cast<const float4*>(sxs);
            const bool mine = p.glu ? col < p.out.n_out : n < p.N;
            int v[8];
            int c = c_lo + half * 8;
            if (c < c_hi) tmem_ld8(acc_at + (uint32_t)c, v);
#pragma unroll 1
            for (; c < c_hi; c += 16, sx4 += 2) {
                const float4 s0 = sx4[0], s1 = sx4[1];
                const float sx[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                int u[8];
                tmem_there(v);
#pragma unroll
                for (int j = 0; j < 8; j++) u[j] = v[j];
                if (c + 16 < c_hi) tmem_ld8(acc_at + (uint32_t)(c + 16), v);
#pragma unroll 1
                for (int k = 0; k < (int)ranks - 1; k++)
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const int4 o = *reinterpret_cast<const int4*>(sums + (size_t)(k * share + c - c_lo + j) * CH + ch * 4);
                        u[j] += o.x; u[j + 1] += o.y; u[j + 2] += o.z; u[j + 3] += o.w;
                    }
                if (!p.glu) {
                    float* y = static_cast<float*>(p.out.y) + (size_t)(m0 + c) * p.out.ldy + n;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float r = finish8(u[j], sx[j] * sw, bias, p.out.cap);
                        if (mine && c + j < c_hi) *y = r;
                        y += p.out.ldy;
                    }
                } else {
                    // 16 gate lanes, 16 up lanes: of two tokens, the lower lanes finish the first and the upper ones the second
                    __nv_bfloat16* f = static_cast<__nv_bfloat16*>(p.out.y) + (size_t)(m0 + c + up) * p.out.ldy + col;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float a = (float)u[j] * (sx[j] * sw), e = (float)u[j + 1] * (sx[j + 1] * sw), other = __shfl_xor_sync(0xffffffffu, up ? a : e, 16);
                        const float r = glu8(p.out.act, up ? other : a, up ? e : other);
                        if (mine && c + j + up < c_hi) *f = __float2bfloat16_rn(r);
                        f += 2 * p.out.ldy;
                    }
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) arrive_first(acc_empty(b));
                else mbar_arrive(acc_empty(b));
            }
        }
    }
    if (ranks > 1 && warp < 2) {                       // (the barriers of the sums)
        __syncwarp();
        whole_cluster();
        whole_cluster();
    }
    tmem_fence_before();
    __syncthreads();
    if (PAIR) whole_cluster();                         // nobody reads or arrives there any more
    if (warp == 1) {
        tmem_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * acc)) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * acc)) : "memory");
    }
}

struct Shape8 { int NX, ranks; bool pair; };

int encode_blocks(CUtensorMap* map, const void* base, long rows, int blocks, int ld, int box_rows) {
    EncodeTiledFn fn;
    const int rc = get_encoder(&fn);
    if (rc) return rc;
    const cuuint64_t dims[3] = {BK8 / 2, (cuuint64_t)rows, (cuuint64_t)blocks}, strides[2] = {(cuuint64_t)ld, BK8};       // two codes an element
    const cuuint32_t box[3] = {BK8 / 2, (cuuint32_t)box_rows, BLOCKS}, one[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CMLB_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with %d for [%ld, %d], stride %d", (int)r, rows, blocks * BK8, ld);
    return CMLB200_OK;
}

// Cycles that a form would take, by its waves: a stage takes its MMAs (4 NX) or its bytes (50 a cycle and SM) or its issue (600), a tile about 2,000 to start and end and 8 a token, a
// cluster's sum 2,000 and 8 a token more. How many clusters of 4 and 8 run at once goes by how SMs lie in groups: 33 and 15 on B200. Tokens are cut into the fewest tiles that hold them, or
// up to three more, which may fill the last wave better. What the two forms that are seldom chosen gain over the best of the others: single CTAs, for a few hundred columns, 27 rows of 54x67 4.1 us (4.6), 157 of
// 332x86 4.75 (5.3), 40 of 32000x64 6.25 (6.6), 3,517 of 2618x360 16.5 (18.0), though 1,081 of 7530x50 14.3 (13.7); clusters of two 41 rows of 5161x13999 19.7 (22.4), 84 of 4405x18379 25.0 (29.8), 32 of 6250x1964
// 7.35 (7.4), though 180 of 4265x4423 12.0 (11.8).
Shape8 pick_shape(int M, int N, int loads) {
    const int sms = cmlb_num_sms(), fewest = (M + 255) / 256;
    auto stage = [](int nx, int rows) { return fmax(fmax(4.0 * nx, BLOCKS * (A8 + rows * BK8) / 50.0), 600.0); };
    auto waves = [](long tiles, int at_once) { return (double)((tiles + at_once - 1) / at_once); };
    const long tn = (N + CH - 1) / CH, tn2 = (N + 2 * CH - 1) / (2 * CH);
    Shape8 best = {};
    double least = 1e300;
    for (int tm = fewest; tm <= fewest + 3; tm++) {
        const int per = (M + tm - 1) / tm, nx = (per + 15) / 16 * 16, nx2 = (per + 31) / 32 * 32;
        auto take = [&](double cost, const Shape8& s) { if (cost < least) { least = cost; best = s; } };
        take(waves(tm * tn, sms) * (loads * stage(nx, nx) + 2000 + 8 * nx), {nx, 1, false});
        take(waves(tm * tn2, sms / 2) * (loads * stage(nx2, nx2 / 2) + 2000 + 8 * nx2), {nx2, 1, true});
        for (int ranks = 2; ranks <= 8 && ranks <= loads; ranks *= 2)
            take(waves(tm * tn, ranks == 2 ? sms / 2 : ranks == 4 ? sms * 33 / 148 : sms * 15 / 148) * ((loads + ranks - 1) / ranks * stage(nx, nx) + 4000 + 16 * nx), {nx, ranks, false});
    }
    return best;
}

template <bool PAIR>
int launch_gemm8(const cmlb200_dense8* W, const int8_t* xq, int ldq, int M, const Shape8& shape, const Out8& out, int glu, int* status, cudaStream_t st) {
    const int blocks = (W->cols + BK8 - 1) / BK8, tm = (M + shape.NX - 1) / shape.NX, rows = PAIR ? 2 * CH : CH, tiles = tm * ((W->rows + rows - 1) / rows), box = PAIR ? shape.NX / 2 : shape.NX;
    CUtensorMap xmap, wmap;
    int rc = encode_blocks(&xmap, xq, M, blocks, ldq, box);
    if (!rc) rc = encode_blocks(&wmap, W->w, W->rows, blocks, W->ld, CH);
    if (rc) return rc;
    const int stage = BLOCKS * (A8 + box * BK8), sums = shape.ranks > 1 ? (shape.NX + 8 * shape.ranks) * CH * 4 : 0;
    const int stages = ROOM8 / stage < MOST_STAGES ? ROOM8 / stage : MOST_STAGES;
    const Gemm8 p = {out, M, W->rows, (blocks + BLOCKS - 1) / BLOCKS, shape.NX, tm, tiles, stages, glu, status};
    const size_t smem = 1024 + HEAD8 + (size_t)(stages * stage > sums ? stages * stage : sums);
    static size_t attr[kMaxDevices] = {};
    CMLB_CUDA(cmlb_ensure_smem(gemm_dense8_kernel<PAIR>, 1024 + HEAD8 + ROOM8, attr));
    const int cluster = PAIR ? 2 : shape.ranks, at_once = cmlb_num_sms() / (PAIR ? 2 : 1);
    const int groups = shape.ranks > 1 || tiles < at_once ? tiles : at_once;
    CMLB_CUDA(launch_chain(gemm_dense8_kernel<PAIR>, dim3((unsigned)(groups * cluster)), dim3(THREADS8), smem, cluster, st, xmap, wmap, p));
    return CMLB200_OK;
}

StatusWords<kMaxDevices> g_status_words8;
int status_word8(int** word) {
    int dev = 0;
    CMLB_CUDA(cudaGetDevice(&dev));
    CMLB_REQUIRE(dev >= 0 && dev < kMaxDevices, "device %d", dev);
    CMLB_CUDA(g_status_words8.get(dev, word));
    return CMLB200_OK;
}

}  // namespace

int cmlb_gemm_dense8(const cmlb200_dense8* W, const int8_t* xq, int ldq, int M, const Out8& out, int glu, cudaStream_t st) {
    int* status;
    const int rc = status_word8(&status);
    if (rc) return rc;
    const Shape8 shape = pick_shape(M, W->rows, (W->cols + BLOCKS * BK8 - 1) / (BLOCKS * BK8));
    return shape.pair ? launch_gemm8<true>(W, xq, ldq, M, shape, out, glu, status, st) : launch_gemm8<false>(W, xq, ldq, M, shape, out, glu, status, st);
}

extern "C" int cmlb200_dense8_status(int* status, int reset) {
    CMLB_REQUIRE(status, "cmlb200_dense8_status: NULL argument");
    int* word;
    const int rc = status_word8(&word);
    if (rc) return rc;
    *status = *static_cast<volatile int*>(word);
    if (reset) *static_cast<volatile int*>(word) = 0;
    return CMLB200_OK;
}
