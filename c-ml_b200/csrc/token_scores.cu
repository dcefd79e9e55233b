// Log probabilities of given tokens, entropy, and the best alternatives of rows of logits.
//
//   m = max x, S = sum of the others' e^(x - m), Q = sum e^(x - m) (x - m):   log p_t = (x_t - m) - ln(1 + S),   H = ln(1 + S) - Q / (1 + S)
//
// S is not below 0 and Q not above, so neither result cancels, no log probability is above 0 and no entropy below, and a row of one value has exactly 0 for both. A row is
// read once, in 16-byte pieces, by a cluster of 1 to 8 CTAs (more for fewer rows). A thread carries both sums in fp32, the largest value's term among them, relative to a
// reference that its warp shares and that follows the warp's largest value at a distance: it moves only when a value is above it by more than 1. At the end of the pass the
// term of the warp's largest value, which is known to the bit, is taken out, and what is left is brought to that value. Q and all exponents are in
// units of ln 2, so a value costs one multiply-add, one exponential and, two values an instruction, its part of both sums. Values where that
// would overflow or lose digits (masked ones, the type's lowest, references beyond a million) are told apart by a round's range and take a longer way. Threads, warps, CTAs and clusters join in a fixed order.
//
// The alternatives need no second pass over the row. A thread remembers the largest of its pieces; the k-th largest of the
// maxima of the CTA's groups of eight threads is a bound that at least k values reach, and few threads hold anything that does. Their pieces are read
// again (from L1 or L2) and what reaches the bound is collected and ranked by counting. Order: value, then lowest index; as keys, the value's
// bits made monotonic above the index's complement. Should more be collected than there is room for (rows whose large values crowd in a
// few threads' pieces), the k best are picked one after the other from the same pieces.
//
// Many rows are bound by the bytes of the logits and the exponentials beside them, few by the chain of barriers behind the pass. Measured: 2,000 rows of 128,000 bf16
// 91.5 us (5.6 TB/s; 57 us are exponentials at 16 a clock and SM), 700 of 128,000 fp32 61.8 us (5.8 TB/s), 256 of 32,000 fp32 with the best 20 15.2 us (10.1 without),
// one of 32,000 with the best 5 5.6 us. Requesting pieces a round ahead cost more registers, and so CTAs under way, than it gave (2,000 rows: 98 to 115 us).
#include <type_traits>

#include "lm_util.cuh"
#include "pairs.cuh"

namespace {

constexpr float kLn2 = 0.693147180559945f;
constexpr int TS_MOST = 32, TS_ROOM = 1024;

typedef uint64_t u64;

// monotonic in the value; 0 is below everything that can be wanted
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);                  // (the two zeros tie)
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ u64 key_of(float v, uint32_t index) { return v > -INFINITY ? ((u64)order_bits(v) << 32) | ~index : 0ull; }

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ void widen_piece(const uint4& u, float (&x)[kPer<T>]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            __half2 t;
            memcpy(&t, &w[i], 4);
            const float2 f = __half22float2(t);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
// largest and smallest of a piece (NaN aside); 16-bit values two at a time
template <typename T> __device__ __forceinline__ void range_of(const uint4& u, float& most, float& least) {
    if constexpr (sizeof(T) == 4) {
        const float a = __uint_as_float(u.x), b = __uint_as_float(u.y), c = __uint_as_float(u.z), d = __uint_as_float(u.w);
        most = fmaxf(fmaxf(a, b), fmaxf(c, d));
        least = fminf(fminf(a, b), fminf(c, d));
    } else {
        typedef std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162> T2;
        T2 t[4];
        memcpy(t, &u, 16);
        const T2 hi = __hmax2(__hmax2(t[0], t[1]), __hmax2(t[2], t[3])), lo = __hmin2(__hmin2(t[0], t[1]), __hmin2(t[2], t[3]));
        most = widen(__hmax(hi.x, hi.y));
        least = widen(__hmin(lo.x, lo.y));
    }
}
__device__ __forceinline__ uint4 ld_row(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// A part of a row: its largest value m, and S and Q of all the others relative to it (no S where there are none, never below zero; Q, in units of ln 2, never
// above). The largest value's own term is exactly 1 and 0 and is not in them, so a part of one value has S = Q = 0.
struct Sums { float m, s, q; };
__device__ __forceinline__ float warp_max(float v) { float m; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v)); return m; }
// what the parts of every `lanes` lanes in turn (a power of two) have together, where those of all such sets of lanes are the same. The first lane that has the largest
// value keeps it out; the other lanes' largest values are values like any other.
template <int lanes>
__device__ __forceinline__ Sums join(const Sums& a) {
    const int lane = (threadIdx.x & 31) & (lanes - 1);
    const float m = warp_max(a.m), d = fmaxf(a.m - m, -1e4f) * kLog2e, c = ex2(d);            // (nothing anywhere: c = 0, and NaN in s stays)
    const int owner = __ffs(__ballot_sync(0xffffffffu, a.m == m)) - 1;
    float s = a.s + (lane == owner || a.m == -INFINITY ? 0.f : 1.f), q = c * fmaf(d, s, a.q);
    s *= c;
#pragma unroll
    for (int o = lanes / 2; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    return {m, s, q};
}

constexpr float TS_TAME = 1048576.f;                   // references up to here: what fl(ref log2(e)) is off by stays below 2^-3
constexpr float TS_LEAST = -1e37f;                     // values down to here: their products with log2(e) do not overflow
constexpr float TS_LAZY = 1.f;                         // the reference moves when a value is above it by more than this, so exponents are below 1.5 and lose no digits of Q

// S and Q of a thread's values, relative to a reference that its warp's threads share. The exponent of a value is x log2(e) - fl(ref log2(e)), one rounding; `shift` is what
// the second product's rounding moved the reference by, and is put right when the reference moves.
struct Running {
    float ref = -INFINITY, minus = 0.f, shift = 0.f;
    u64 s = 0ull, q = 0ull;
    __device__ __forceinline__ bool tame() const { return fabsf(ref) <= TS_TAME; }
    __device__ __forceinline__ void move(float to) {
        const float d = fmaxf(ref - to, -1e4f) * kLog2e - shift;
        ref = to;
        minus = tame() ? -(to * kLog2e) : 0.f;
        shift = tame() ? fmaf(to, kLog2e, minus) : 0.f;
        const float by = d + shift, c = ex2(by);                             // exponents grow by that
        const u64 c2 = pair_of(c, c), d2 = pair_of(by, by);
        q = fma_pair(c2, fma_pair(d2, s, q), 0ull);
        s = fma_pair(c2, s, 0ull);
    }
    // of any value; of one at or above TS_LEAST the fast way finds the same bits
    __device__ __forceinline__ float exponent(float x) const { return tame() ? fmaf(x, kLog2e, minus) : (x - (ref == -INFINITY ? 0.f : ref)) * kLog2e; }
    // values beside masked ones, or as large as numbers get
    __device__ __forceinline__ void take_wild(float x) {
        const float t = exponent(x), e = ex2(t);
        s = add_pair(s, pair_of(e, 0.f));
        q = fma_pair(pair_of(e, 0.f), pair_of(fmaxf(t, -1e4f), 0.f), q);
    }
    // The warp's part, `most` being this thread's largest value. What the largest of all put into the sums is taken out again, to the bit (it was met under the present
    // reference: only a larger value could have moved that since); what rounding leaves on the wrong side of zero is nothing.
    __device__ __forceinline__ Sums sums(float most) const {
        const int lane = threadIdx.x & 31;
        const float m = warp_max(most);
        const int owner = __ffs(__ballot_sync(0xffffffffu, most == m)) - 1;
        float s0, s1, q0, q1;
        unpair(s, s0, s1);
        unpair(q, q0, q1);
        float ss = s0 + s1, qq = q0 + q1;
        const float t = exponent(m);
        if (lane == owner && m > -INFINITY) {
            const float e = ex2(t);
            ss -= e;
            qq -= __fmul_rn(e, t);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            qq += __shfl_xor_sync(0xffffffffu, qq, o);
        }
        if (m == -INFINITY) return {m, ss, qq};        // (nothing, or NaN)
        const float c = ex2(-t);
        qq = c * fmaf(-t, ss, qq);
        ss *= c;
        return {m, ss < 0.f ? 0.f : ss, qq > 0.f ? 0.f : qq};
    }
};
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// grid = rows * splits, clusters of `splits`.
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS)
token_scores_kernel(const T* __restrict__ logits, long ld, int vocab, const int* __restrict__ tokens, int top, int splits, float* __restrict__ logprob, float* __restrict__ entropy,
                    int* __restrict__ top_ids, float* __restrict__ top_logprob) {
    constexpr int PER = kPer<T>, WARPS = THREADS / 32, GROUPS = THREADS / 8;
    static_assert(GROUPS >= TS_MOST, "every group's best could be wanted");
    __shared__ Sums w_sums[WARPS], c_sums[8];
    __shared__ u64 g_best[GROUPS], bound, room[TS_ROOM], c_best[8 * TS_MOST], last_room[8 * TS_MOST], w_best[WARPS];
    __shared__ uint8_t holders[WARPS][32];
    __shared__ int num_room, num_last;
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (met below: the cluster's CTAs have begun)
    dep_wait();
    dep_trigger();
    const int rank = blockIdx.x % splits, r = blockIdx.x / splits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* row = logits + (size_t)r * ld;
    // the row: `head` values up to a 16-byte boundary, `pieces` of 16 bytes, `tail` values; this CTA's pieces are lo .. hi - 1
    const int head = min(vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T)), pieces = (vocab - head) / PER, tail = vocab - head - pieces * PER;
    const int per = (pieces + splits - 1) / splits, lo = min(pieces, rank * per), hi = min(pieces, lo + per);
    const T* body = row + head;
    Running a;
    float best = -INFINITY;                            // largest value, and the number of its piece
    uint32_t best_piece = 0;
    auto note = [&](float most, uint32_t piece) {
        if (most > best) { best = most; best_piece = piece; }
    };
    // all of a warp come here, before they take values of which this thread's largest is `most`
    auto prepare = [&](float most) {
        if (__any_sync(0xffffffffu, most > a.ref + TS_LAZY)) a.move(fmaxf(a.ref, warp_max(most)));
    };
    auto take = [&](const uint4& u, bool fast) {
        float x[PER];
        widen_piece<T>(u, x);
        if (fast) {
            const u64 unit = pair_of(kLog2e, kLog2e), minus = pair_of(a.minus, a.minus);
#pragma unroll
            for (int i = 0; i < PER; i += 2) {
                const u64 t = fma_pair(pair_of(x[i], x[i + 1]), unit, minus);
                float t0, t1;
                unpair(t, t0, t1);
                const u64 e = pair_of(ex2(t0), ex2(t1));
                a.s = add_pair(a.s, e);
                a.q = fma_pair(e, t, a.q);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) a.take_wild(x[i]);
        }
    };
    // numbers of pieces ascend along the row: head values, pieces, tail values
    auto single = [&](int i) { return i < head ? (uint32_t)i : (uint32_t)(head + pieces + i); };
    auto take_one = [&](bool on, const T* at, int i) {
        const float x = on ? widen(*at) : -INFINITY;
        note(x, single(i));
        prepare(x);
        if (on) a.take_wild(x);
    };
    if (rank == 0 && warp * 32 < head) take_one((int)threadIdx.x < head, row + threadIdx.x, threadIdx.x);
    // Four pieces a thread and round, a warp's threads together; the last round has what is left
    auto round = [&](int v, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        uint4 u[4];
        float most = -INFINITY, least = INFINITY;      // one masked value sends all of the round the longer way
#pragma unroll
        for (int j = 0; j < 4; j++) if (WHOLE || v + j * THREADS < hi) u[j] = ld_row(body + (size_t)(v + j * THREADS) * PER);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (WHOLE || v + j * THREADS < hi) {
                float m, l;
                range_of<T>(u[j], m, l);
                if (!WHOLE) note(m, (uint32_t)(head + v + j * THREADS));
                most = fmaxf(most, m);
                least = fminf(least, l);
            }
        if (WHOLE && most > best) {                    // (seldom)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (TOP) {
                    float m, l;
                    range_of<T>(u[j], m, l);
                    note(m, (uint32_t)(head + v + j * THREADS));
                }
            best = most;
        }
        prepare(most);
        const bool fast = least >= TS_LEAST && a.tame();
#pragma unroll
        for (int j = 0; j < 4; j++) if (WHOLE || v + j * THREADS < hi) take(u[j], fast);
    };
    int v = lo + warp * 32;
    for (; v + 3 * THREADS + 32 <= hi; v += 4 * THREADS) round(v + lane, std::true_type());
    if (v < hi) round(v + lane, std::false_type());
    if (rank == splits - 1 && warp * 32 < tail) take_one((int)threadIdx.x < tail, body + (size_t)pieces * PER + threadIdx.x, head + threadIdx.x);
    const Sums w_part = a.sums(best);
    if (lane == 0) w_sums[warp] = w_part;
    const u64 mine = TOP ? key_of(best, best_piece) : 0ull;
    if (TOP) {
        u64 g = mine;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) { const u64 x = __shfl_xor_sync(0xffffffffu, g, o); g = x > g ? x : g; }
        if ((lane & 7) == 0) g_best[threadIdx.x >> 3] = g;
        if (threadIdx.x == 0) { bound = 1ull; num_room = 0; num_last = 0; }
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        const Sums none = {-INFINITY, 0.f, 0.f}, t = join<32>(lane < WARPS ? w_sums[lane] : none);
        const uint32_t dst = cluster_addr(&c_sums[rank], 0);
        if (lane == 0) {
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(t.m) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(t.s) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(t.q) : "memory");
        }
    }
    if (TOP) {
        // the bound: the top-th largest of the groups' best, or nothing where fewer have any. A group's threads share the comparing
        const u64 g = g_best[threadIdx.x >> 3];
        int above = 0;
#pragma unroll
        for (int i = 0; i < GROUPS / 8; i++) above += g_best[8 * i + (lane & 7)] > g;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (g && above == top - 1) bound = g;          // (all of a group's threads have found the same)
        __syncthreads();
        const u64 floor_ = bound;
        const uint32_t hit = __ballot_sync(0xffffffffu, mine >= floor_);
        const int ns = __popc(hit), most = (hi - lo + THREADS - 1) / THREADS;        // pieces of a thread, and its head and tail value
        if (mine >= floor_) holders[warp][__popc(hit & ((1u << lane) - 1))] = (uint8_t)lane;
        __syncwarp();
        // calls f(value, index, piece) for what the warp's threads that hold anything went through
        auto again = [&](auto f) {
            for (int i = lane; i < ns * (most + 2); i += 32) {
                const int j = i / ns, t = warp * 32 + holders[warp][i - j * ns];
                if (j < most) {
                    const int w = lo + t + j * THREADS;
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
        const uint32_t dst = cluster_addr(&c_best[rank * top], 0);
        if (nr <= TS_ROOM) {
            for (int i = threadIdx.x; i < nr; i += THREADS) {
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
                for (int w = 0; w < WARPS; w++) next = w_best[w] > next ? w_best[w] : next;
                last = next;
                if (threadIdx.x == 0) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * n), "l"(next) : "memory");
            }
        }
    }
    if (splits > 1) cluster_sync();
    else __syncthreads();
    if (rank) return;                                  // (nobody reads another CTA's memory from here on)
    const Sums none = {-INFINITY, 0.f, 0.f}, t = join<8>((lane & 7) < splits ? c_sums[lane & 7] : none);
    const bool nothing = t.m == -INFINITY && t.s == 0.f;
    const float ls = log1pf(t.s);                      // (t.s is not below 0, so no log probability is above it)
    if (threadIdx.x == 0) {
        if (logprob) {
            const int id = tokens[r];
            logprob[r] = nothing || id < 0 || id >= vocab ? -INFINITY : (widen(row[id]) - t.m) - ls;
        }
        if (entropy) entropy[r] = nothing ? 0.f : ls - t.q / (1.f + t.s) * kLn2;
    }
    if (TOP) {
        // what each CTA of the cluster found is in order; nothing below any CTA's last can be wanted
        const int n = splits * top;
        u64 least = 0ull;
        for (int i = 0; i < splits; i++) { const u64 k = c_best[i * top + top - 1]; least = k > least ? k : least; }
        for (int i = threadIdx.x; i < n; i += THREADS)
            if (c_best[i] && c_best[i] >= least) last_room[atomicAdd(&num_last, 1)] = c_best[i];
        __syncthreads();
        const int found = num_last;
        for (int i = threadIdx.x; i < max(found, top); i += THREADS) {
            const u64 k = i < found ? last_room[i] : 0ull;
            int above = i < found ? 0 : i;             // (places without a value come last)
            for (int j = 0; i < found && j < found; j++) above += last_room[j] > k;
            if (above >= top) continue;
            const size_t at = (size_t)r * top + above;
            if (top_ids) top_ids[at] = k ? (int)~(uint32_t)k : -1;
            if (top_logprob) top_logprob[at] = k ? (order_value((uint32_t)(k >> 32)) - t.m) - ls : -INFINITY;
        }
    }
}

template <typename T>
int launch_scores(const void* d_logits, long ld, int rows, int vocab, const int* d_tokens, int top, float* d_logprob, float* d_entropy, int* d_top_ids, float* d_top_logprob, cudaStream_t st) {
    // A cluster's CTAs read at least 8 KB each; more of them share a row while every one has an SM of its own (64 rows of 50,000 bf16, best 20: 8.3 us by
    // two each, 9.5 by one, 11.1 by four)
    int splits = 1;
    while (splits < 8 && (long long)rows * splits * 2 <= cmlb_num_sms() && (size_t)vocab * sizeof(T) > (size_t)splits * 8192) splits *= 2;
    // Many short rows are a matter of how many CTAs are under way, not of how fast each is: 256 threads for those (2,000 rows of 1,000, best 5: 15.7 us, with
    // 512 threads 27.0; 256 rows of 32,000, best 20: 19.0 and 15.4)
    const bool small = (long long)rows >= 4 * cmlb_num_sms() && (size_t)vocab * sizeof(T) <= 65536;
    const dim3 grid((unsigned)rows * splits);
    auto run = [&](auto kernel, int threads) {
        return launch_chain(kernel, grid, dim3(threads), 0, splits, st, (const T*)d_logits, ld, vocab, d_tokens, top, splits, d_logprob, d_entropy, d_top_ids, d_top_logprob);
    };
    if (top) CMLB_CUDA(small ? run(token_scores_kernel<T, true, 256>, 256) : run(token_scores_kernel<T, true, 512>, 512));
    else CMLB_CUDA(small ? run(token_scores_kernel<T, false, 256>, 256) : run(token_scores_kernel<T, false, 512>, 512));
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
