// Drafted tokens against the target's logits, and tokens drawn on the device.
//
//   p = softmax(l / T), q = softmax(l' / T) of the drafter (or 1 at the draft). Draft i is kept while u_i q(d_i) < p(d_i). The token behind the kept ones is drawn from p
//   where all were kept, else from max(p - q, 0): the token with the largest w_j / E_j, E_j = -ln(1 - v_j), w the weights up to a factor.
//
// E are standard exponentials, so the first of them to "arrive" at rates w is token j with probability w_j / sum w: no running sums along the vocabulary, whose
// rounding would move every border between tokens, one maximum that may be taken in any order, and no second pass for the sum. All random numbers come out of Philox4x32-10
// (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011) keyed by the sequence's 64-bit number: v of token j is word j mod 4 of
// counter (j / 4, 0, 0, 0), u_i word i mod 4 of counter (i / 4, 1, 0, 0).
//
// Two launches. draft_stats: the rows that drafts are tested against, several CTAs a row: largest value and sum of exponentials, fp32 in a thread and fp64 between threads (or, for
// greedy sequences, the place of the largest). draft_token: a cluster a sequence finds the first draft that is turned down, and draws over the one row (and the drafter's)
// that counts: in fp32 first, then the CTA's candidates within what that can be off by again in fp64, so that which token is drawn does not hang on the order of anything.
#include <type_traits>

#include "lm_util.cuh"

namespace {

constexpr int VS_THREADS = 256, VT_THREADS = 512, VS_SPLITS = 16;
constexpr float kGreedy = 1e-5f;                       // colder is greedy

struct Stat { float most; int at; double sum; };       // of a part of a row: largest value, its first place (greedy), sum of e^((x - most) / T)

struct Philox { uint32_t w[4]; };
__device__ __forceinline__ Philox philox(uint64_t key, uint32_t c0, uint32_t c1) {
    uint32_t a = c0, b = c1, c = 0u, d = 0u, k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t m0 = (uint64_t)a * 0xD2511F53u, m1 = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(m1 >> 32) ^ b ^ k0;
        c = (uint32_t)(m0 >> 32) ^ d ^ k1;
        b = (uint32_t)m1;
        d = (uint32_t)m0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{a, b, c, d}};
}
__device__ __forceinline__ float lg2(float v) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// log2 of -ln(1 - v), v = (word + 1/2) / 2^32, to about 1e-4: by the series where 1 - v has lost digits of v
__device__ __forceinline__ float log_wait(uint32_t word) {
    const float v = ((float)word + 0.5f) * 2.3283064365386963e-10f, rest = ((float)~word + 0.5f) * 2.3283064365386963e-10f;
    return lg2(v < 0.0625f ? v * fmaf(v, fmaf(v, 0.33333334f, 0.5f), 1.f) : lg2(rest) * -0.6931471805599453f);
}
// ln of the same
__device__ __forceinline__ double log_wait_exact(uint32_t word) { return log(-log1p(-((double)word + 0.5) * 2.3283064365386963e-10)); }

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ void widen_piece(const uint4& u, float (&x)[kPer<T>]) {
    T t[kPer<T>];
    memcpy(t, &u, 16);
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) x[i] = widen(t[i]);
}
// lowest place of the largest value; NaN (as such) above everything, so that a row with it is known
__device__ __forceinline__ void better(float& v, int& at, float v2, int at2) {
    if (v2 > v || (v2 == v && at2 < at)) { v = v2; at = at2; }
}

struct Verify {
    cmlb200_drafts d;
    long ld;
    int vocab;
};

// Part `split` of target row (which = 0) or drafter's row (1) of draft i. grid = drafts * sides * splits.
template <typename T>
__global__ void __launch_bounds__(VS_THREADS)
draft_stats_kernel(const Verify v, const T* __restrict__ logits, int sides, int splits, Stat* __restrict__ stats) {
    __shared__ int mine;
    __shared__ Stat parts[VS_THREADS / 32];
    dep_trigger();
    dep_wait();
    const int split = blockIdx.x % splits, side = blockIdx.x / splits % sides, i = blockIdx.x / splits / sides, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) mine = -1;
    __syncthreads();
    // the sequence that draft i belongs to: drafts of s are first[s] - s .. first[s + 1] - s - 2
    for (int s = threadIdx.x; s < v.d.sequences; s += VS_THREADS)
        if (v.d.first[s] - s <= i && i < v.d.first[s + 1] - s - 1) mine = s;
    __syncthreads();
    const int s = mine;
    if (s < 0) return;                                 // (rows that no sequence has)
    const float heat = v.d.temperature ? v.d.temperature[s] : 1.f;
    const bool greedy = !(heat >= kGreedy);
    if (greedy && side) return;
    const T* row = side ? static_cast<const T*>(v.d.logits) + (size_t)i * v.d.ld : logits + (size_t)(i + s) * v.ld;
    constexpr int PER = kPer<T>;
    const int V = v.vocab, head = min(V, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T)), pieces = (V - head) / PER, tail = V - head - pieces * PER;
    const int per = (pieces + splits - 1) / splits, lo = min(pieces, split * per), hi = min(pieces, lo + per);
    const T* body = row + head;
    const float c = greedy ? 0.f : __fdiv_rn(kLog2e, heat);
    float most = -INFINITY, sum = 0.f;
    int at = 0;
    auto raise = [&](float to) {
        if (to > most) {
            sum *= ex2((most - to) * c);               // (from -inf: 0 times 0)
            most = to;
        }
    };
    auto one = [&](float x, int place) {
        if (greedy) {
            if (x > most) { most = x; at = place; }
            if (x != x) sum = x;
        } else {
            raise(x);
            if (x != -INFINITY) sum += ex2((x - most) * c);
        }
    };
    if (split == 0 && (int)threadIdx.x < head) one(widen(row[threadIdx.x]), threadIdx.x);
    constexpr int U = 4;
    for (int p0 = lo + threadIdx.x; p0 < hi; p0 += U * VS_THREADS) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; j++)
            if (p0 + j * VS_THREADS < hi) u[j] = *reinterpret_cast<const uint4*>(body + (size_t)(p0 + j * VS_THREADS) * PER);
#pragma unroll
        for (int j = 0; j < U; j++) {
            if (p0 + j * VS_THREADS >= hi) break;
            float x[PER];
            widen_piece<T>(u[j], x);
            if (greedy) {
#pragma unroll
                for (int e = 0; e < PER; e++) one(x[e], head + (p0 + j * VS_THREADS) * PER + e);
            } else {
                float m = x[0];
#pragma unroll
                for (int e = 1; e < PER; e++) m = fmaxf(m, x[e]);
                raise(m);
                const float ref = most == -INFINITY ? 0.f : most;          // (a NaN still shows)
#pragma unroll
                for (int e = 0; e < PER; e++) sum += ex2((x[e] - ref) * c);
            }
        }
    }
    if (split == splits - 1 && (int)threadIdx.x < tail) one(widen(body[(size_t)pieces * PER + threadIdx.x]), head + pieces * PER + threadIdx.x);
    auto join = [&](Stat a, const Stat& b) {
        Stat r = a;
        better(r.most, r.at, b.most, b.at);
        if (greedy) r.sum = a.sum + b.sum;
        else r.sum = (a.most == -INFINITY ? a.sum : a.sum * (double)ex2((a.most - r.most) * c)) + (b.most == -INFINITY ? b.sum : b.sum * (double)ex2((b.most - r.most) * c));
        return r;
    };
    Stat a = {most, at, (double)sum};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stat b = {__shfl_xor_sync(0xffffffffu, a.most, o), __shfl_xor_sync(0xffffffffu, a.at, o), __shfl_xor_sync(0xffffffffu, a.sum, o)};
        a = join(a, b);
    }
    if (lane == 0) parts[warp] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < VS_THREADS / 32; k++) a = join(a, parts[k]);
        stats[((size_t)i * sides + side) * splits + split] = a;
    }
}

// A row's parts together. most = +inf or a sum that is not a number: no distribution
__device__ __forceinline__ Stat whole_row(const Stat* parts, int splits, bool greedy, double rate) {
    Stat a = parts[0];
    for (int k = 1; k < splits; k++) better(a.most, a.at, parts[k].most, parts[k].at);
    double sum = 0.0;
    for (int k = 0; k < splits; k++)
        sum += greedy || parts[k].most == -INFINITY ? parts[k].sum : parts[k].sum * exp(((double)parts[k].most - (double)a.most) * rate);
    a.sum = sum;
    return a;
}
__device__ __forceinline__ bool holds(const Stat& a) { return a.most > -INFINITY && a.most < INFINITY && a.sum == a.sum; }

// grid = sequences * ranks, clusters of `ranks` (up to 8)
template <typename T>
__global__ void __launch_bounds__(VT_THREADS)
draft_token_kernel(const Verify v, const T* __restrict__ logits, int sides, int splits, const Stat* __restrict__ stats, int ranks, int* __restrict__ accepted, int* __restrict__ next) {
    struct Best { double z; int at; int bad; };
    __shared__ int stop_at;
    __shared__ float2 w_most[VT_THREADS / 32];
    __shared__ Best w_best[VT_THREADS / 32], c_best[8];
    dep_trigger();
    dep_wait();
    const int rank = blockIdx.x % ranks, s = blockIdx.x / ranks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, V = v.vocab;
    const int first = v.d.first[s], end = v.d.first[s + 1];
    if (first < s || end <= first || end - (s + 1) > v.d.rows - v.d.sequences) {       // not a sequence's rows (all of a cluster's CTAs see the same)
        if (rank == 0 && threadIdx.x == 0) { accepted[s] = 0; next[s] = -1; }
        return;
    }
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (met below: the cluster's CTAs have begun)
    const int n = end - first - 1;
    const float heat = v.d.temperature ? v.d.temperature[s] : 1.f;
    const bool greedy = !(heat >= kGreedy);
    const double rate = greedy ? 0.0 : 1.0 / (double)heat;
    const uint64_t key = v.d.random ? v.d.random[s] : 0ull;
    const int draft0 = first - s;
    if (threadIdx.x == 0) stop_at = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += VT_THREADS) {
        const int token = v.d.tokens[draft0 + i];
        bool kept = token >= 0 && token < V;
        if (kept) {
            const Stat* at = stats + (size_t)(draft0 + i) * sides * splits;
            const Stat p = whole_row(at, splits, greedy, rate);
            if (!holds(p)) kept = false;
            else if (greedy) kept = p.at == token;
            else {
                const double chance = exp(((double)widen(logits[(size_t)(first + i) * v.ld + token]) - (double)p.most) * rate) / p.sum;
                double q = 1.0;
                if (sides > 1) {
                    const Stat b = whole_row(at + splits, splits, false, rate);
                    if (holds(b)) q = exp(((double)widen(static_cast<const T*>(v.d.logits)[(size_t)(draft0 + i) * v.d.ld + token]) - (double)b.most) * rate) / b.sum;
                }
                kept = (double)philox(key, (uint32_t)i >> 2, 1u).w[i & 3] * 2.3283064365386963e-10 * q < chance;
            }
        }
        if (!kept) atomicMin(&stop_at, i);
    }
    __syncthreads();
    const int stop = stop_at;
    const T* row = logits + (size_t)(first + stop) * v.ld;
    // what is taken off: the drafter's chances, or the draft itself
    const T* less = nullptr;
    int without = -1;
    float p_most = 0.f, q_most = 0.f, p_unit = 1.f, q_unit = 0.f;
    double p_sum = 1.0, q_sum = 1.0;
    if (stop < n && !greedy) {
        const Stat* at = stats + (size_t)(draft0 + stop) * sides * splits;
        if (sides > 1) {
            const Stat b = whole_row(at + splits, splits, false, rate);
            if (holds(b)) {
                const Stat p = whole_row(at, splits, false, rate);
                less = static_cast<const T*>(v.d.logits) + (size_t)(draft0 + stop) * v.d.ld;
                p_most = p.most; q_most = b.most;
                p_sum = p.sum; q_sum = b.sum;
                p_unit = (float)(1.0 / p.sum); q_unit = (float)(1.0 / b.sum);
            }
        }
        if (!less) without = v.d.tokens[draft0 + stop];
    }
    const float c = greedy ? 1.f : __fdiv_rn(kLog2e, heat);
    const int groups = (V + 3) / 4, per = (groups + ranks - 1) / ranks, lo = rank * per, hi = min(groups, lo + per);
    for (int pass = 0;; pass++) {
        // log2 of w / E of every token, and the thread's best. Where w is p alone: relative to the largest logit that the thread has met, so that logits far from zero lose no digits
        float most = -INFINITY, ref = less || greedy ? 0.f : -INFINITY;
        int at = 0x7fffffff, bad = 0;
        for (int g = lo + threadIdx.x; g < hi; g += VT_THREADS) {
            Philox r;
            if (!greedy) r = philox(key, (uint32_t)g, 0u);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = 4 * g + e;
                if (j >= V) break;
                const float x = widen(row[j]);
                if (!(x < INFINITY)) bad = 1;
                float z;
                if (greedy) z = x;
                else if (less) {
                    const float w = ex2((x - p_most) * c) * p_unit - ex2((widen(less[j]) - q_most) * c) * q_unit;
                    z = w > 0.f ? lg2(w) - log_wait(r.w[e]) : -INFINITY;
                } else {
                    if (x > ref) {
                        most += (ref - x) * c;         // (nothing yet: -inf)
                        ref = x;
                    }
                    z = j == without ? -INFINITY : (x - ref) * c - log_wait(r.w[e]);           // (-inf beside -inf: NaN, which is never the best)
                }
                if (z > most) { most = z; at = j; }
            }
        }
        auto raise = [&](float& r, float& m, float r2, float m2) {
            const float top = fmaxf(r, r2);
            m = fmaxf(m > -INFINITY ? m + (r - top) * c : m, m2 > -INFINITY ? m2 + (r2 - top) * c : m2);
            r = top;
        };
        float top = ref, m = most;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) raise(top, m, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) w_most[warp] = make_float2(top, m);
        __syncthreads();
        top = w_most[0].x;
        m = w_most[0].y;
#pragma unroll
        for (int k = 1; k < VT_THREADS / 32; k++) raise(top, m, w_most[k].x, w_most[k].y);
        // candidates again, in 64 bits
        Best b = {-INFINITY, at, bad};
        if (most > -INFINITY) {
            if (greedy) b.z = (double)most;
            else if (most + (ref - top) * c >= m - (2e-3f + fabsf(m) * 1e-5f)) {
                double w;
                if (less) {
                    const double d = exp(((double)widen(row[at]) - (double)p_most) * rate) / p_sum - exp(((double)widen(less[at]) - (double)q_most) * rate) / q_sum;
                    w = d > 0.0 ? log(d) : -1e30;              // (what 32 bits took for a weight was their rounding)
                } else w = (double)widen(row[at]) * rate;
                b.z = w - log_wait_exact(philox(key, (uint32_t)at >> 2, 0u).w[at & 3]);
            }
        }
        auto join = [](Best& a, const Best& o) {
            if (o.z > a.z || (o.z == a.z && o.at < a.at)) { a.z = o.z; a.at = o.at; }
            a.bad |= o.bad;
        };
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Best x = {__shfl_xor_sync(0xffffffffu, b.z, o), __shfl_xor_sync(0xffffffffu, b.at, o), __shfl_xor_sync(0xffffffffu, b.bad, o)};
            join(b, x);
        }
        if (lane == 0) w_best[warp] = b;
        if (pass == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        __syncthreads();
        if (warp == 0) {
            b = lane < VT_THREADS / 32 ? w_best[lane] : Best{-INFINITY, 0x7fffffff, 0};
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) {
                const Best x = {__shfl_xor_sync(0xffffffffu, b.z, o), __shfl_xor_sync(0xffffffffu, b.at, o), __shfl_xor_sync(0xffffffffu, b.bad, o)};
                join(b, x);
            }
            // every CTA of the cluster learns of every one's best
            if (lane < ranks) {
                const uint32_t dst = cluster_addr(&c_best[rank], lane);
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dst), "d"(b.z) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 8), "r"(b.at) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 12), "r"(b.bad) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        Best all = c_best[0];
        for (int k = 1; k < ranks; k++) join(all, c_best[k]);
        // where rounding leaves nothing of p - q (or p is nothing but the draft), p itself
        const bool again = pass == 0 && !all.bad && all.z == -INFINITY && (less || without >= 0);
        if (!again) {
            if (rank == 0 && threadIdx.x == 0) {
                accepted[s] = stop;
                next[s] = all.bad || all.z == -INFINITY ? -1 : all.at;
            }
            return;
        }
        less = nullptr;
        without = -1;
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");      // nobody reads what the next pass writes
    }
}

template <typename T>
int launch_verify(const Verify& v, const void* logits, int* accepted, int* next, void* work, cudaStream_t st) {
    const int drafts = v.d.rows - v.d.sequences, sides = v.d.logits ? 2 : 1;
    Stat* stats = static_cast<Stat*>(work);
    int splits = 1;
    while (splits < VS_SPLITS && (long)drafts * sides * splits * 2 <= 4l * cmlb_num_sms() && (size_t)v.vocab * sizeof(T) > (size_t)splits * 8192) splits *= 2;
    if (drafts)
        CMLB_CUDA(launch_chain(draft_stats_kernel<T>, dim3((unsigned)((long)drafts * sides * splits)), dim3(VS_THREADS), 0, 1, st, v, static_cast<const T*>(logits), sides, splits, stats));
    int ranks = 1;
    while (ranks < 8 && (long)v.d.sequences * ranks * 2 <= 2l * cmlb_num_sms() && v.vocab > ranks * 2048) ranks *= 2;
    CMLB_CUDA(launch_chain(draft_token_kernel<T>, dim3((unsigned)(v.d.sequences * ranks)), dim3(VT_THREADS), 0, ranks, st, v, static_cast<const T*>(logits), sides, splits, (const Stat*)stats, ranks,
                           accepted, next));
    return CMLB200_OK;
}

}  // namespace

extern "C" size_t cmlb200_verify_work_bytes(int rows, int sequences) {
    if (sequences <= 0 || rows < sequences) return 0;
    return (size_t)(rows - sequences + 1) * 2 * VS_SPLITS * sizeof(Stat);
}

extern "C" int cmlb200_verify_drafts(const cmlb200_drafts* d, const void* d_logits, int dtype, long ld, int vocab, int* d_accepted, int* d_next, void* d_work, void* stream) {
    static const char* who = "cmlb200_verify_drafts";
    CMLB_REQUIRE(d && d_logits && d_accepted && d_next && d_work && d->first, "%s: NULL argument", who);
    CMLB_REQUIRE(d->sequences > 0 && d->rows >= d->sequences && d->rows <= (1 << 20), "%s: %d rows of %d sequences", who, d->rows, d->sequences);
    CMLB_REQUIRE(vocab > 0 && ld >= vocab && (!d->logits || d->ld >= vocab), "%s: %d logits, strides %ld and %ld", who, vocab, ld, d->ld);
    CMLB_REQUIRE(d->tokens || d->rows == d->sequences, "%s: %d drafts without tokens", who, d->rows - d->sequences);
    CMLB_REQUIRE(d->random || d->temperature, "%s: no random numbers, and no temperatures that could do without", who);
    CMLB_REQUIRE((((uintptr_t)d_logits | (uintptr_t)d->logits) & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0 && ((uintptr_t)d_work & 15) == 0 && ((uintptr_t)d->random & 7) == 0,
                 "%s: pointers are not aligned to their types (workspace: 16 bytes)", who);
    const Verify v = {*d, ld, vocab};
    cudaStream_t st = as_stream(stream);
    if (dtype == CMLB200_DT_F32) return launch_verify<float>(v, d_logits, d_accepted, d_next, d_work, st);
    if (dtype == CMLB200_DT_BF16) return launch_verify<__nv_bfloat16>(v, d_logits, d_accepted, d_next, d_work, st);
    if (dtype == CMLB200_DT_F16) return launch_verify<__half>(v, d_logits, d_accepted, d_next, d_work, st);
    CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    return CMLB200_EINVAL;
}
