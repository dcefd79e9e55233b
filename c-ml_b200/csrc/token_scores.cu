// Log probabilities of given tokens, entropy, and the best alternatives of rows of logits.
//
//   m = max x, S = sum e^(x - m), Q = sum e^(x - m) (x - m):   log p_t = x_t - m - ln S,   H = ln S - Q / S
//
// Both parts of H are positive, so nothing cancels. A row is read once, in 16-byte pieces, by a cluster of 1 to 8 CTAs (more for
// fewer rows); m, S and Q are carried in fp32 and meet in a fixed order: warp, CTA, cluster. Bound by the bytes of the logits.
//
// The alternatives need no second pass over the row. A thread remembers the largest of its pieces; the k-th largest of the
// maxima of the CTA's groups of eight threads is a bound that at least k values reach, and few threads hold anything that does. Their pieces are read
// again (from L2) and what reaches the bound is collected and ranked by counting. Order: value, then lowest index; as keys, the value's
// bits made monotonic above the index's complement. Should more be collected than there is room for (rows whose large values crowd in a
// few threads' pieces), the k best are picked one after the other from the same pieces.
#include "lm_util.cuh"

namespace {

constexpr int TS_THREADS = 512, TS_WARPS = TS_THREADS / 32, TS_GROUPS = TS_THREADS / 8, TS_MOST = 32, TS_ROOM = 1024;
static_assert(TS_GROUPS >= TS_MOST, "every group's best could be wanted");

typedef unsigned long long u64;

// monotonic in the value; 0 is below everything that can be wanted
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);                  // (the two zeros tie)
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ u64 key_of(float v, uint32_t index) { return v > -INFINITY ? ((u64)order_bits(v) << 32) | ~index : 0ull; }

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ void widen_piece(const uint4& u, float (&x)[kPer<T>]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            T t[2];
            memcpy(t, &w[i], 4);
            x[2 * i] = widen(t[0]);
            x[2 * i + 1] = widen(t[1]);
        }
    }
}
__device__ __forceinline__ uint4 ld_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

struct Sums { float m, s, q; };
// what two disjoint parts of a row have together
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s, a.q + b.q};                     // (NaN in s stays)
    const float da = fmaxf(a.m - m, -1e30f), db = fmaxf(b.m - m, -1e30f), ca = __expf(da), cb = __expf(db);
    return {m, a.s * ca + b.s * cb, ca * (a.q + da * a.s) + cb * (b.q + db * b.s)};
}
__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// grid = rows * splits, clusters of `splits`.
template <typename T, bool TOP>
__global__ void __launch_bounds__(TS_THREADS)
token_scores_kernel(const T* __restrict__ logits, long ld, int vocab, const int* __restrict__ tokens, int top, int splits, float* __restrict__ logprob, float* __restrict__ entropy,
                    int* __restrict__ top_ids, float* __restrict__ top_logprob) {
    constexpr int PER = kPer<T>;
    __shared__ Sums w_sums[TS_WARPS], c_sums[8];
    __shared__ u64 g_best[TS_GROUPS], bound, room[TS_ROOM], best[8 * TS_MOST], w_best[TS_WARPS];
    __shared__ int stripes[TS_THREADS], num_stripes, num_room;
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (met below: the cluster's CTAs have begun)
    dep_wait();
    dep_trigger();
    const int rank = blockIdx.x % splits, r = blockIdx.x / splits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* row = logits + (size_t)r * ld;
    // the row: `head` values up to a 16-byte boundary, `pieces` of 16 bytes, `tail` values; this CTA's pieces are lo .. hi - 1
    const int head = min(vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T)), pieces = (vocab - head) / PER, tail = vocab - head - pieces * PER;
    const int per = (pieces + splits - 1) / splits, lo = min(pieces, rank * per), hi = min(pieces, lo + per);
    const T* body = row + head;
    Sums a = {-INFINITY, 0.f, 0.f};
    u64 mine = 0ull;                                   // largest piece: its value's bits above the complement of its number
    // n values whose piece has the number `piece` (a single value of head or tail is a piece of its own)
    auto take = [&](const float* x, int n, uint32_t piece) {
        float g = x[0];
        for (int i = 1; i < n; i++) g = fmaxf(g, x[i]);
        if (TOP) { const u64 k = key_of(g, piece); mine = k > mine ? k : mine; }
        if (g > a.m) {
            const float d = fmaxf(a.m - g, -1e30f), c = __expf(d);
            a.q = c * (a.q + d * a.s);
            a.s *= c;
            a.m = g;
        }
        const float m = a.m == -INFINITY ? 0.f : a.m;
        for (int i = 0; i < n; i++) {
            const float d = x[i] - m, e = ex2(d * kLog2e);
            a.s += e;
            a.q = fmaf(e, fmaxf(d, -1e4f), a.q);
        }
    };
    // numbers of pieces ascend along the row: head values, pieces, tail values
    auto single = [&](int i) { return i < head ? (uint32_t)i : (uint32_t)(head + pieces + i); };
    const bool has_head = rank == 0 && (int)threadIdx.x < head, has_tail = rank == splits - 1 && (int)threadIdx.x < tail;
    if (has_head) { const float x = widen(row[threadIdx.x]); take(&x, 1, single(threadIdx.x)); }
    int v = lo + threadIdx.x;
    for (; v + 3 * TS_THREADS < hi; v += 4 * TS_THREADS) {
        uint4 u[4];
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = ld_once(body + (size_t)(v + j * TS_THREADS) * PER);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x[PER];
            widen_piece<T>(u[j], x);
            take(x, PER, (uint32_t)(head + v + j * TS_THREADS));
        }
    }
    for (; v < hi; v += TS_THREADS) {
        float x[PER];
        widen_piece<T>(ld_once(body + (size_t)v * PER), x);
        take(x, PER, (uint32_t)(head + v));
    }
    if (has_tail) { const float x = widen(body[(size_t)pieces * PER + threadIdx.x]); take(&x, 1, single(head + threadIdx.x)); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = join(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.q, o)});
    if (lane == 0) w_sums[warp] = a;
    if (TOP) {
        u64 g = mine;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) { const u64 x = __shfl_xor_sync(0xffffffffu, g, o); g = x > g ? x : g; }
        if ((lane & 7) == 0) g_best[threadIdx.x >> 3] = g;
        if (threadIdx.x == 0) { bound = 1ull; num_stripes = 0; num_room = 0; }
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        Sums t = w_sums[0];
#pragma unroll
        for (int w = 1; w < TS_WARPS; w++) t = join(t, w_sums[w]);
        const uint32_t dst = remote(&c_sums[rank], 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(t.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(t.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(t.q) : "memory");
    }
    if (TOP) {
        if (threadIdx.x < TS_GROUPS) {                 // the bound: the top-th largest of the groups' best, or nothing where fewer have any
            const u64 k = g_best[threadIdx.x];
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < TS_GROUPS; i++) above += g_best[i] > k;
            if (k && above == top - 1) bound = k;
        }
        __syncthreads();
        if (mine >= bound) stripes[atomicAdd(&num_stripes, 1)] = threadIdx.x;
        __syncthreads();
        const int ns = num_stripes, most = (hi - lo + TS_THREADS - 1) / TS_THREADS;        // pieces of a thread, and its head and tail value
        const u64 floor_ = bound;
        // calls f(value, index, piece) for what the listed threads went through
        auto again = [&](auto f) {
            for (int i = threadIdx.x; i < ns * (most + 2); i += TS_THREADS) {
                const int j = i / ns, t = stripes[i - j * ns];
                if (j < most) {
                    const int w = lo + t + j * TS_THREADS;
                    if (w >= hi) continue;
                    float x[PER];
                    widen_piece<T>(*reinterpret_cast<const uint4*>(body + (size_t)w * PER), x);
#pragma unroll
                    for (int e = 0; e < PER; e++) f(x[e], head + w * PER + e, (uint32_t)(head + w));
                } else if (j == most) {
                    if (rank == 0 && t < head) f(widen(row[t]), t, single(t));
                } else if (rank == splits - 1 && t < tail) {
                    f(widen(body[(size_t)pieces * PER + t]), head + pieces * PER + t, single(head + t));
                }
            }
        };
        again([&](float x, int index, uint32_t piece) {
            if (key_of(x, piece) < floor_) return;
            const int at = atomicAdd(&num_room, 1);
            if (at < TS_ROOM) room[at] = key_of(x, (uint32_t)index);
        });
        __syncthreads();
        const int nr = num_room;
        const uint32_t dst = remote(&best[rank * top], 0);
        if (nr <= TS_ROOM) {
            for (int i = threadIdx.x; i < nr; i += TS_THREADS) {
                const u64 k = room[i];
                int above = 0;
                for (int j = 0; j < nr; j++) above += room[j] > k;
                if (above < top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * above), "l"(k) : "memory");
            }
            if ((int)threadIdx.x >= nr && (int)threadIdx.x < top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * threadIdx.x), "l"(0ull) : "memory");
        } else {
            u64 last = ~0ull;
            for (int n = 0; n < top; n++) {
                u64 next = 0ull;
                again([&](float x, int index, uint32_t) { const u64 k = key_of(x, (uint32_t)index); if (k < last && k > next) next = k; });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) { const u64 x = __shfl_xor_sync(0xffffffffu, next, o); next = x > next ? x : next; }
                __syncthreads();
                if (lane == 0) w_best[warp] = next;
                __syncthreads();
                for (int w = 0; w < TS_WARPS; w++) next = w_best[w] > next ? w_best[w] : next;
                last = next;
                if (threadIdx.x == 0) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * n), "l"(next) : "memory");
            }
        }
    }
    if (splits > 1) cluster_sync();
    else __syncthreads();
    if (rank) return;                                  // (nobody reads another CTA's memory from here on)
    Sums t = c_sums[0];
    for (int s = 1; s < splits; s++) t = join(t, c_sums[s]);
    const bool nothing = t.m == -INFINITY && t.s == 0.f;
    const float ls = logf(t.s);
    if (threadIdx.x == 0) {
        if (logprob) {
            const int id = tokens[r];
            logprob[r] = nothing || id < 0 || id >= vocab ? -INFINITY : (widen(row[id]) - t.m) - ls;
        }
        if (entropy) entropy[r] = nothing ? 0.f : ls - t.q / t.s;
    }
    if (TOP)
        for (int i = threadIdx.x; i < splits * top; i += TS_THREADS) {
            const u64 k = best[i];
            int above = 0;
            for (int j = 0; j < splits * top; j++) above += best[j] > k || (best[j] == k && j < i);        // (only places without a value are equal)
            if (above >= top) continue;
            const size_t at = (size_t)r * top + above;
            if (top_ids) top_ids[at] = k ? (int)~(uint32_t)k : -1;
            if (top_logprob) top_logprob[at] = k ? (order_value((uint32_t)(k >> 32)) - t.m) - ls : -INFINITY;
        }
}

template <typename T>
int launch_scores(const void* d_logits, long ld, int rows, int vocab, const int* d_tokens, int top, float* d_logprob, float* d_entropy, int* d_top_ids, float* d_top_logprob, cudaStream_t st) {
    // a cluster's CTAs read at least 8 KB each: more of them while rows are fewer than two CTAs an SM
    int splits = 1;
    while (splits < 8 && (long long)rows * splits < 2 * cmlb_num_sms() && (size_t)vocab * sizeof(T) > (size_t)splits * 8192) splits *= 2;
    const dim3 grid((unsigned)rows * splits);
    if (top) CMLB_CUDA(launch_chain(token_scores_kernel<T, true>, grid, dim3(TS_THREADS), 0, splits, st, (const T*)d_logits, ld, vocab, d_tokens, top, splits, d_logprob, d_entropy, d_top_ids, d_top_logprob));
    else CMLB_CUDA(launch_chain(token_scores_kernel<T, false>, grid, dim3(TS_THREADS), 0, splits, st, (const T*)d_logits, ld, vocab, d_tokens, top, splits, d_logprob, d_entropy, d_top_ids, d_top_logprob));
    return CMLB200_OK;
}

}  // namespace

extern "C" int cmlb200_token_scores(const void* d_logits, int dtype, long ld, int rows, int vocab, const int* d_tokens, int top, float* d_logprob, float* d_entropy, int* d_top_ids,
                                    float* d_top_logprob, void* stream) {
    static const char* who = "cmlb200_token_scores";
    CMLB_REQUIRE(d_logits && rows > 0 && vocab > 0 && ld >= vocab, "%s: %d rows of %d logits, stride %ld", who, rows, vocab, ld);
    CMLB_REQUIRE(rows <= (1 << 27), "%s: %d rows", who, rows);
    CMLB_REQUIRE(top >= 0 && top <= TS_MOST && top <= vocab && (top == 0 || d_top_ids || d_top_logprob), "%s: the best %d of %d (up to %d, and somewhere to put them)", who, top, vocab, TS_MOST);
    CMLB_REQUIRE(!d_logprob == !d_tokens, "%s: tokens and their log probabilities go together", who);
    CMLB_REQUIRE(top || d_logprob || d_entropy, "%s: nothing is asked for", who);
    CMLB_REQUIRE(((uintptr_t)d_logits & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0, "%s: logits are not aligned to their type", who);
    cudaStream_t st = as_stream(stream);
    if (dtype == CMLB200_DT_F32) return launch_scores<float>(d_logits, ld, rows, vocab, d_tokens, top, d_logprob, d_entropy, d_top_ids, d_top_logprob, st);
    if (dtype == CMLB200_DT_BF16) return launch_scores<__nv_bfloat16>(d_logits, ld, rows, vocab, d_tokens, top, d_logprob, d_entropy, d_top_ids, d_top_logprob, st);
    if (dtype == CMLB200_DT_F16) return launch_scores<__half>(d_logits, ld, rows, vocab, d_tokens, top, d_logprob, d_entropy, d_top_ids, d_top_logprob, st);
    CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    return CMLB200_EINVAL;
}
