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
// Two launches. draft_stats: the rows that drafts are tested against, several CTAs a row: sums of exponentials in fp32, 16 or 32 values at a time (or, for greedy sequences, the place of the largest).
// draft_token: a cluster a sequence finds the first draft that is turned down, and draws over the one row (and the drafter's) that counts, in fp32. What fp32 cannot tell is decided in fp64, sums of the
// rows included, so that neither hangs on the order of anything: u q and p that lie closer than the sums are sure; a best token that is not above all others by more than they can be off by, where a
// token of p - q, which may lose all its digits, has a least and a most. It is seldom, and kept out of the way of the loops: 5 to 11 us more for a draw over 32,000 or
// 128,000 tokens, 12 to 26 with a drafter's row.
// Measured: four drafts of one sequence over 32,000 tokens 9.2 us, of 32 sequences over 128,000 41.7 (22.5 for the bytes: 25 for the tested rows, the rest for the draws, which are some 45 instructions a token,
// a third of them Philox, on 256 CTAs), one draw over 32,000 5.0, 64 over 128,000 21.0 (with one loop for all kinds of rows: 22.6).
// Few rows are bound by the chain of dependent loads and by code that is fetched anew with every launch (hence small loops, and what is seldom needed out of the way), many by memory.
#include <atomic>
#include <type_traits>

#include "lm_util.cuh"

namespace {

constexpr int VS_THREADS = 256, VT_THREADS = 512, VS_SPLITS = 16, MOST_RANKS = 16;
constexpr float kGreedy = 1e-5f;                       // colder is greedy
constexpr float kClose = 0.998f;
// What two chances from 32-bit exponentials may be off by together, relative to themselves: an exponential 2^-22 and 2^-23 of its exponent (142 at most); a row's sum 4e-6 for that (of exponents
// that are 30 at most where they weigh anything), 2e-6 for 32 values added, 3e-6 for parts put together three times, and 2^-24 for each of a thread's 32 values or more, of which there are V / 4096 at
// most. Closer calls are decided in 64 bits.
__device__ __forceinline__ double doubt_of(int vocab) { return 3.0517578125e-5 + 2.9103830456733704e-11 * (double)vocab; }
constexpr float kLazy = 16.f;                          // a reference is changed where a value is 2^16 times as large
constexpr int MOST_VOCAB = 1 << 28;
// (infinite ones would make no number of the logits of tokens that cannot come; no number at all stays that, which is greedy)
__device__ __forceinline__ float heat_of(const cmlb200_drafts& d, int s) {
    const float t = d.temperature ? d.temperature[s] : 1.f;
    return t > 1e30f ? 1e30f : t;
}

// Of a part of a row: largest value and its first place (greedy), or a value that none is far above, the draft's logit and the sum of e^((x - most) / T). A sum that is not a number:
// the part holds NaN or +inf
struct Stat { float most; int at; float sum; int pad; };
static_assert(VS_SPLITS <= 16, "a row's parts are put together by half a warp");

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
// v = (word + 1/2) / 2^32 to 2^-23 of itself
__device__ __forceinline__ float uniform_of(uint32_t word) { return fmaf((float)word, 2.3283064365386963e-10f, 1.1641532e-10f); }
// -ln(1 - v): the first terms of its series, which are never above it, and to about 1e-4 of itself
__device__ __forceinline__ float least_wait(float v) { return v * fmaf(v, fmaf(v, 0.33333334f, 0.5f), 1.f); }
// (1 - v from the word's complement, which is as exact next to 1 as v is next to 0)
__device__ __forceinline__ float wait_of(uint32_t word) {
    const float v = uniform_of(word);
    return v < 0.0625f ? least_wait(v) : lg2(uniform_of(~word)) * -0.6931471805599453f;
}
// u of draft i
__device__ __forceinline__ double coin(uint64_t key, int i) { return (double)philox(key, (uint32_t)i >> 2, 1u).w[i & 3] * 2.3283064365386963e-10; }
__device__ __noinline__ double far_log(double v) { return log(v); }
__device__ __noinline__ double far_exp(double v) { return exp(v); }
// ln of the same: 1 - v is exact in 64 bits
__device__ __forceinline__ double log_wait_exact(uint32_t word) { return far_log(-far_log(((double)~word + 0.5) * 2.3283064365386963e-10)); }

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ void widen_piece(const uint4& u, float (&x)[kPer<T>]) {
    T t[kPer<T>];
    memcpy(t, &u, 16);
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) x[i] = widen(t[i]);
}
template <typename T> __device__ __forceinline__ T lowest();                 // a logit of a token that cannot come
template <> __device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xfc00); }
__device__ __forceinline__ float max_nan(float a, float b) { float m; asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b)); return m; }
__device__ __forceinline__ float warp_max(float v) { float m; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v)); return m; }

__device__ __forceinline__ double lane_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
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
    const float heat = heat_of(v.d, s);
    const bool greedy = !(heat >= kGreedy);
    if (greedy && side) return;
    const T* row = side ? static_cast<const T*>(v.d.logits) + (size_t)i * v.d.ld : logits + (size_t)(i + s) * v.ld;
    constexpr int PER = kPer<T>;
    // pieces of 16 bytes as they lie in memory; the first and the last may begin or end outside the row
    const int V = v.vocab, lead = (int)(((uintptr_t)row & 15) / sizeof(T)), pieces = (lead + V + PER - 1) / PER, per = (pieces + splits - 1) / splits, lo = split * per, hi = min(pieces, lo + per);
    const float c = greedy ? 0.f : __fdiv_rn(kLog2e, heat);
    float most = -INFINITY, sum = 0.f;
    int at = 0;
    constexpr int U = 4;
#pragma unroll 1
    for (int p0 = lo + threadIdx.x; p0 < hi; p0 += U * VS_THREADS) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int e0 = (p0 + j * VS_THREADS) * PER - lead;
            if (p0 + j * VS_THREADS >= hi) break;
            if (e0 >= 0 && e0 + PER <= V) u[j] = *reinterpret_cast<const uint4*>(row + e0);
            else {
                T t[PER];
#pragma unroll
                for (int e = 0; e < PER; e++) t[e] = e0 + e >= 0 && e0 + e < V ? row[e0 + e] : lowest<T>();
                memcpy(&u[j], t, 16);
            }
        }
        if (greedy) {
#pragma unroll
            for (int j = 0; j < U; j++) {
                if (p0 + j * VS_THREADS >= hi) break;
                float x[PER];
                widen_piece<T>(u[j], x);
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    if (x[e] > most) { most = x[e]; at = (p0 + j * VS_THREADS) * PER - lead + e; }
                    if (x[e] != x[e]) sum = x[e];
                }
            }
            continue;
        }
        float part = 0.f;                              // of 16 or 32 values
#pragma unroll
        for (int j = 0; j < U; j++) {
            if (p0 + j * VS_THREADS >= hi) break;
            float x[PER];
            widen_piece<T>(u[j], x);
            float m = x[0];
#pragma unroll
            for (int e = 1; e < PER; e++) m = fmaxf(m, x[e]);
            if ((m - most) * c > kLazy) {              // (what was there before weighs 2^-16 at most, and so does what its factor is off by)
                const float by = ex2((most - m) * c);  // (from -inf: 0 times 0)
                sum *= by;
                part *= by;
                most = m;
            }
            const float ref = most == -INFINITY ? 0.f : most;                  // (a NaN still shows)
#pragma unroll
            for (int e = 0; e < PER; e++) part += ex2((x[e] - ref) * c);
        }
        sum += part;
    }
    // the warp's part, then the CTA's
    auto together = [&]() {
        const float top = warp_max(most);
        if (greedy) {
            at = (int)__reduce_min_sync(0xffffffffu, most == top ? (uint32_t)at : 0xffffffffu);
        } else if (most > -INFINITY) sum *= ex2((most - top) * c);
        most = top;
        sum = lane_sum(sum);
    };
    together();
    if (lane == 0) parts[warp] = {most, at, sum, 0};
    __syncthreads();
    if (warp) return;
    const Stat mine_ = lane < VS_THREADS / 32 ? parts[lane] : Stat{-INFINITY, 0x7fffffff, 0.f, 0};
    most = mine_.most;
    at = mine_.at;
    sum = mine_.sum;
    together();
    if (lane == 0) {
        if (!greedy && split == 0) {
            const int token = v.d.tokens[i];
            at = __float_as_int(token >= 0 && token < V ? widen(row[token]) : -INFINITY);
        }
        stats[((size_t)i * sides + side) * splits + split] = {most, at, sum, 0};
    }
}

// What a draft was tested against, from the parts: the target's row by the lower half of a warp, the drafter's by the upper one
struct Tested { Stat p, q; };
__device__ __forceinline__ Tested tested(const Stat* parts, int sides, int splits, float c, bool greedy) {
    const int lane = threadIdx.x & 31, side = lane >> 4, k = lane & 15;
    Stat a = {-INFINITY, 0x7fffffff, 0.f, 0};
    if (side < sides && k < splits) a = parts[side * splits + k];
    float top = a.most;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    int at = greedy ? (a.most == top ? a.at : 0x7fffffff) : __shfl_sync(0xffffffffu, a.at, lane & 16);
    float sum = greedy || a.most == -INFINITY ? a.sum : a.sum * ex2((a.most - top) * c);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (greedy) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
    }
    return {{__shfl_sync(0xffffffffu, top, 0), __shfl_sync(0xffffffffu, at, 0), __shfl_sync(0xffffffffu, sum, 0), 0},
            {__shfl_sync(0xffffffffu, top, 16), __shfl_sync(0xffffffffu, at, 16), __shfl_sync(0xffffffffu, sum, 16), 0}};
}
__device__ __forceinline__ bool holds(const Stat& a) { return a.most > -INFINITY && a.most < INFINITY && a.sum == a.sum; }

__device__ __forceinline__ void cluster_all() { asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// What a cluster's CTAs tell one another where 64 bits decide
struct Weighed {
    double best[VT_THREADS / 32 + MOST_RANKS];
    int at[VT_THREADS / 32 + MOST_RANKS];
    double warps[VT_THREADS / 32], sums[2][MOST_RANKS];
};
// Sum of e^((x - from) rate) over a row that holds numbers, in 64 bits throughout, by a cluster together, in an order that is always the same. Two calls one after another are turn 0 and turn 1
template <typename T> __device__ __noinline__ double exact_sum(const T* row, int vocab, double from, double rate, int ranks, int turn, Weighed* in) {
    const int rank = blockIdx.x % ranks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, end = (int)((long)vocab * (rank + 1) / ranks);
    double sum = 0.0;
#pragma unroll 2
    for (int j = (int)((long)vocab * rank / ranks) + threadIdx.x; j < end; j += VT_THREADS) sum += exp(((double)widen(row[j]) - from) * rate);
    sum = lane_sum64(sum);
    __syncthreads();
    if (lane == 0) in->warps[warp] = sum;
    __syncthreads();
    sum = lane_sum64(lane < VT_THREADS / 32 ? in->warps[lane] : 0.0);
    if (warp == 0 && lane < ranks) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(&in->sums[turn][rank], lane)), "d"(sum) : "memory");
    cluster_all();                                     // (and all have read what the turn before the last left)
    return lane_sum64(lane < ranks ? in->sums[turn][lane] : 0.0);
}

// What the best of some tokens has at most and at least, and the most that any of the others has, as logarithms to the base 2 relative to a logit `ref` times c; the best's token, the lowest of equals
struct Best { float z, least, others, ref; int at, bad; };
// of a warp's lanes together
__device__ __forceinline__ Best best_of_lanes(Best b, float c) {
    const float top = warp_max(b.ref), by = b.ref == top ? 0.f : (b.ref - top) * c;
    const float z = b.z + by, most = warp_max(z);      // (-inf where there is nothing)
    const int at = (int)__reduce_min_sync(0xffffffffu, z == most ? (uint32_t)b.at : 0xffffffffu);
    const bool it = z == most && b.at == at;           // (a token is one lane's)
    return {most, warp_max(it ? b.least + by : -INFINITY), warp_max(fmaxf(it ? -INFINITY : z, b.others + by)), top, at, (int)__reduce_or_sync(0xffffffffu, (unsigned)b.bad)};
}
// the largest of four but number `but`
__device__ __forceinline__ float most_but(const float (&x)[4], int but) {
    return fmaxf(fmaxf(but == 0 ? -INFINITY : x[0], but == 1 ? -INFINITY : x[1]), fmaxf(but == 2 ? -INFINITY : x[2], but == 3 ? -INFINITY : x[3]));
}
// logits of tokens 4 g .. 4 g + 3; whole: rows lie on boundaries of four
template <typename T> __device__ __forceinline__ void load4(const T* row, int g, int vocab, bool whole, float (&x)[4]) {
    if (whole && 4 * g + 4 <= vocab) {
        T t[4];
        if constexpr (sizeof(T) == 4) { const uint4 u = *reinterpret_cast<const uint4*>(row + 4 * (size_t)g); memcpy(t, &u, 16); }
        else { const uint2 u = *reinterpret_cast<const uint2*>(row + 4 * (size_t)g); memcpy(t, &u, 8); }
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = widen(t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = 4 * g + e < vocab ? widen(row[4 * (size_t)g + e]) : -INFINITY;
    }
}

constexpr int KEPT = 32;                               // drafts whose rows' parts are kept put together
__device__ __forceinline__ double chance(const Stat& a, double rate) { return far_exp(((double)__int_as_float(a.at) - (double)a.most) * rate); }
// What is asked for seldom is worked out anew from memory, out of the way of the loops: held for it, things would have no registers there.
__device__ __forceinline__ uint64_t key_of(const cmlb200_drafts& d, int s) { return d.random ? d.random[s] : 0ull; }
// The first draft that is turned down, from number `from` on, or their number: with sums in 64 bits throughout where u q and p lie closer than their rows' sums are sure. A cluster together
template <typename T>
__device__ __noinline__ int settle(const Verify& v, const T* logits, const Stat* stats, int splits, int ranks, int from, Weighed* in) {
    const int s = blockIdx.x / ranks, first = v.d.first[s], n = v.d.first[s + 1] - first - 1, sides = v.d.logits ? 2 : 1;
    const float heat = heat_of(v.d, s), c = __fdiv_rn(kLog2e, heat);
    const double rate = 1.0 / (double)heat;
    for (int i = from; i < n; i++) {
        const int d = first - s + i, token = v.d.tokens[d];
        const Tested t = tested(stats + (size_t)d * sides * splits, sides, splits, c, false);
        if (token < 0 || token >= v.vocab || !holds(t.p)) return i;
        const bool beside = sides > 1 && holds(t.q);
        const double u = coin(key_of(v.d, s), i), p = chance(t.p, rate), q = beside ? chance(t.q, rate) : 1.0, p_near = p / (double)t.p.sum, uq_near = beside ? u * (q / (double)t.q.sum) : u;
        bool kept = uq_near < p_near;
        if (fabs(uq_near - p_near) < doubt_of(v.vocab) * p_near) {
            const double p_sum = exact_sum(logits + (size_t)(first + i) * v.ld, v.vocab, t.p.most, rate, ranks, 0, in);
            const double q_sum = beside ? exact_sum(static_cast<const T*>(v.d.logits) + (size_t)d * v.d.ld, v.vocab, t.q.most, rate, ranks, 1, in) : 1.0;
            kept = u * (q / q_sum) < p / p_sum;
            cluster_all();                             // (turn 0 again)
        }
        if (!kept) return i;
    }
    return n;
}

// A draw behind `stop` drafts whose best tokens lie closer than 32 bits tell: every token of these groups that could be the best is weighed in 64 bits, sums of its rows included. A
// cluster together. kind: 0 p itself, 1 p without the draft, 2 p - q
template <typename T>
__device__ __noinline__ int weigh(const Verify& v, const T* logits, const Stat* stats, int splits, int ranks, int stop, int kind, float ref, float least, Weighed* in) {
    const int rank = blockIdx.x % ranks, s = blockIdx.x / ranks, first = v.d.first[s], d = first - s + stop, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, V = v.vocab;
    const int groups = (V + 3) / 4, per = (groups + ranks - 1) / ranks, lo = rank * per, hi = min(groups, lo + per), without = kind == 1 ? v.d.tokens[d] : -1;
    const float heat = heat_of(v.d, s), c = __fdiv_rn(kLog2e, heat), doubt = (float)doubt_of(V), bound = ex2(least) * (kClose * 2.3283064365386963e-10f);
    const uint64_t key = key_of(v.d, s);
    const double rate = 1.0 / (double)heat;
    const T *row = logits + (size_t)(first + stop) * v.ld, *less = kind == 2 ? static_cast<const T*>(v.d.logits) + (size_t)d * v.d.ld : nullptr;
    Tested t = {};
    double p_sum = 1.0, q_sum = 1.0;
    if (less) {
        t = tested(stats + (size_t)d * 2 * splits, 2, splits, c, false);
        p_sum = exact_sum(row, V, t.p.most, rate, ranks, 0, in);
        q_sum = exact_sum(less, V, t.q.most, rate, ranks, 1, in);
    }
    const float p_unit = (1.f + doubt) / t.p.sum, q_unit = (1.f - doubt) / t.q.sum;
    double z = -INFINITY;
    int token = 0x7fffffff;
#pragma unroll 1
    for (int j = 4 * lo + threadIdx.x; j < min(V, 4 * hi); j += VT_THREADS) {
        const float x = widen(row[j]), y = less ? widen(less[j]) : 0.f;
        const uint32_t word = philox(key, (uint32_t)j >> 2, 0u).w[j & 3];
        const float w = less ? ex2((x - t.p.most) * c) * p_unit - ex2((y - t.q.most) * c) * q_unit : ex2((x - ref) * c);
        if (!(w >= bound * (float)word) || j == without) continue;
        double l;
        if (less) {
            const double e = ((double)x - (double)t.p.most) * rate, p = far_exp(e) / p_sum, more = p - far_exp(((double)y - (double)t.q.most) * rate) / q_sum;
            // (what 64 bits' exponents and sums may be off by: the same distribution from shifted logits is nothing above itself)
            if (!(more > (1.2e-13 + 4.4e-19 * (double)V + 4.5e-16 * fabs(e)) * p)) continue;
            l = far_log(more);
        } else l = ((double)x - (double)ref) * rate;
        l -= log_wait_exact(word);
        if (l > z) { z = l; token = j; }               // (a thread's tokens ascend)
    }
    for (int level = 0; level < 3; level++) {
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) {
            const double z2 = __shfl_xor_sync(0xffffffffu, z, o);
            const int t2 = __shfl_xor_sync(0xffffffffu, token, o);
            if (z2 > z || (z2 == z && t2 < token)) { z = z2; token = t2; }
        }
        if (level == 2) break;
        if (level == 0) {
            __syncthreads();
            if (lane == 0) { in->best[warp] = z; in->at[warp] = token; }
            __syncthreads();
            z = lane < VT_THREADS / 32 ? in->best[lane] : -INFINITY;
            token = lane < VT_THREADS / 32 ? in->at[lane] : 0x7fffffff;
        } else {
            if (warp == 0 && lane < ranks) {
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(&in->best[VT_THREADS / 32 + rank], lane)), "d"(z) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&in->at[VT_THREADS / 32 + rank], lane)), "r"(token) : "memory");
            }
            cluster_all();
            z = lane < ranks ? in->best[VT_THREADS / 32 + lane] : -INFINITY;
            token = lane < ranks ? in->at[VT_THREADS / 32 + lane] : 0x7fffffff;
        }
    }
    return token;
}

// grid = sequences * ranks, clusters of `ranks`. Two CTAs an SM: with more than 64 registers a thread, which leave room for one, 32 sequences of 4 drafts over 128,000 tokens took 56 us instead of 42
template <typename T>
__global__ void __launch_bounds__(VT_THREADS, 2)
draft_token_kernel(const __grid_constant__ Verify v, const T* __restrict__ logits, int sides, int splits, const Stat* __restrict__ stats, int ranks, int* __restrict__ accepted, int* __restrict__ next) {
    __shared__ int stop_at, doubt_at;
    __shared__ Best w_best[VT_THREADS / 32], c_best[MOST_RANKS];
    __shared__ Weighed far;
    __shared__ Tested kept_stats[KEPT];
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
    const float heat = heat_of(v.d, s);
    const bool greedy = !(heat >= kGreedy);
    const double rate = greedy ? 0.0 : 1.0 / (double)heat;
    const float c = greedy ? 0.f : __fdiv_rn(kLog2e, heat);
    uint64_t key = v.d.random ? v.d.random[s] : 0ull;
    // (known to be the same for a warp: its multiples stay in uniform registers)
    key = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(key >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)key);
    const int draft0 = first - s;
    if (threadIdx.x == 0) stop_at = doubt_at = n;
    __syncthreads();
    for (int i = warp; i < n; i += VT_THREADS / 32) {          // a warp a draft
        const int token = v.d.tokens[draft0 + i];
        const Tested t = tested(stats + (size_t)(draft0 + i) * sides * splits, sides, splits, c, greedy);
        if (i < KEPT && lane == 0) kept_stats[i] = t;
        bool kept = token >= 0 && token < V && holds(t.p);
        if (greedy) kept = kept && t.p.at == token;
        else if (kept) {
            const double q = sides > 1 && holds(t.q) ? chance(t.q, rate) / (double)t.q.sum : 1.0, p = chance(t.p, rate) / (double)t.p.sum, uq = coin(key, i) * q;
            kept = uq < p;
            if (fabs(uq - p) < doubt_of(V) * p && lane == 0) atomicMin(&doubt_at, i);
        }
        if (!kept && lane == 0) atomicMin(&stop_at, i);
    }
    __syncthreads();
    int stop = stop_at;
    bool unsettled = doubt_at <= stop && doubt_at < n, plain = false;
    const int groups = (V + 3) / 4, per = (groups + ranks - 1) / ranks, lo = rank * per, hi = min(groups, lo + per);
    bool first_time = true;
    for (;;) {
        const int s = blockIdx.x / ranks, first = v.d.first[s], n = v.d.first[s + 1] - first - 1, draft0 = first - s;
        const T* row = logits + (size_t)(first + stop) * v.ld;
        // what is taken off: the drafter's chances, or the draft itself
        const T* less = nullptr;
        int without = -1;
        Tested t = {};
        if (stop < n && !greedy && !plain) {
            if (sides > 1) {
                t = stop < KEPT ? kept_stats[stop] : tested(stats + (size_t)(draft0 + stop) * sides * splits, sides, splits, c, greedy);
                if (holds(t.q)) less = static_cast<const T*>(v.d.logits) + (size_t)(draft0 + stop) * v.d.ld;
            }
            if (!less) without = v.d.tokens[draft0 + stop];
        }
        // of p - q at most
        const float doubt = (float)doubt_of(V), p_unit = less ? (1.f + doubt) / t.p.sum : 0.f, q_unit = less ? (1.f - doubt) / t.q.sum : 0.f;
        const bool whole = (((uintptr_t)row | (uintptr_t)less) & (4 * sizeof(T) - 1)) == 0;
        // A warp's threads share a bound: the largest weight over wait that any of them has met. A token that comes within kClose of it with v, which is never above its wait, is looked at; there are
        // few, and only for those a wait is worked out. Where w is p alone it is relative to a logit that none that the warp has met is far above, so that logits far from zero lose no digits (greedy: the logits
        // themselves). p - q may lose all of its digits: a token counts with what it is at most, the bound is what the best is at least.
        float best = greedy ? -INFINITY : 0.f, least = 0.f, others = 0.f, bound = 0.f, ref = less || greedy ? 0.f : -INFINITY;
        int at = 0x7fffffff, bad = 0;
        // one loop for each kind of row: none holds registers for another
        auto scan = [&](auto greedy_, auto residual_) {
            constexpr bool GREEDY = decltype(greedy_)::value, RESIDUAL = decltype(residual_)::value;
            constexpr int U = 2;                           // groups of four tokens under way
#pragma unroll 1
            for (int g0 = lo + warp * 32; g0 < hi; g0 += U * VT_THREADS) {
                float x[U][4], y[U][4];
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int g = g0 + k * VT_THREADS + lane;
                    load4(row, g < hi ? g : groups, V, whole, x[k]);               // (behind the end: -inf)
                    if (RESIDUAL) load4(less, g < hi ? g : groups, V, whole, y[k]);
                }
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int g = g0 + k * VT_THREADS + lane;
                    const float most = max_nan(max_nan(x[k][0], x[k][1]), max_nan(x[k][2], x[k][3]));
                    bad |= !(most < INFINITY);
                    if (GREEDY) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (x[k][e] > best) { best = x[k][e]; at = 4 * g + e; }
                        }
                        continue;
                    }
                    const Philox r = philox(key, (uint32_t)g, 0u);
                    float w[4];
                    if (RESIDUAL) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            y[k][e] = ex2((y[k][e] - t.q.most) * c) * q_unit;
                            w[e] = ex2((x[k][e] - t.p.most) * c) * p_unit - y[k][e];
                        }
                    } else {
                        const float top = (uint32_t)(without - 4 * g) < 4u ? most_but(x[k], without - 4 * g) : most;          // (the draft that was turned down sets no reference)
                        if (__any_sync(0xffffffffu, (top - ref) * c > kLazy)) {        // (a best token outlives three such changes at most)
                            const float to = fmaxf(ref, warp_max(top)), by = ref == -INFINITY ? 0.f : ex2((ref - to) * c);
                            best *= by;
                            others *= by;
                            bound *= by;
                            ref = to;
                        }
                        const float from = ref == -INFINITY ? 0.f : ref;
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = ex2((x[k][e] - from) * c);
                        if ((uint32_t)(without - 4 * g) < 4u) {
#pragma unroll
                            for (int e = 0; e < 4; e++) if (4 * g + e == without) w[e] = 0.f;
                        }
                    }
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) any |= w[e] > bound * (float)r.w[e];
                    if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (!(w[e] > bound * (float)r.w[e])) continue;
                            const float arrives = __fdividef(1.f, wait_of(r.w[e])), score = w[e] * arrives;
                            if (score > best) {
                                others = best;
                                best = score;
                                at = 4 * g + e;
                                // (p - q with both off the other way)
                                if (RESIDUAL) least = fmaf(-2.f * doubt * arrives, fmaf(2.f, y[k][e], w[e]), score);
                            } else others = fmaxf(others, score);
                        }
                        bound = warp_max(RESIDUAL ? fmaxf(least, 0.f) : best) * (kClose * 2.3283064365386963e-10f);
                    }
                }
            }
        };
        if (greedy) scan(std::true_type(), std::false_type());
        else if (less) scan(std::false_type(), std::true_type());
        else scan(std::false_type(), std::false_type());
        // thread, CTA and cluster have the best and what the others come to
        const float z = greedy ? best : best > 0.f ? lg2(best) : -INFINITY;
        const Best b = {z, !less ? z : least > 0.f ? lg2(least) : -INFINITY, others > 0.f ? lg2(others) : -INFINITY, ref, at, bad};
        auto best_of = [&](Best x) {
            x = best_of_lanes(x, c);
            if (lane == 0) w_best[warp] = x;
            if (first_time) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            first_time = false;
            __syncthreads();
            const Best none = {-INFINITY, -INFINITY, -INFINITY, less || greedy ? 0.f : -INFINITY, 0x7fffffff, 0};
            if (warp == 0) {
                x = best_of_lanes(lane < VT_THREADS / 32 ? w_best[lane] : none, c);
                if (lane < ranks) {
                    const uint32_t dst = cluster_addr(&c_best[rank], lane);
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(x.z) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(x.least) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(x.others) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 12), "f"(x.ref) : "memory");
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 16), "r"(x.at) : "memory");
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 20), "r"(x.bad) : "memory");
                }
            }
            cluster_all();
            return best_of_lanes(lane < ranks ? c_best[lane] : none, c);
        };
        Best all = best_of(b);
        // What 32 bits are off by at most: 1e-4 of the waits, 1e-5 of logarithms and of products with c (tokens near the best lie within 64 of it). All CTAs know the same: they decide together.
        constexpr float slack = 1e-3f;
        // Differences below 2^-126 are nothing in 32 bits: where the best comes to less than 2^-80 (some of them over a wait of 2^-33), all tokens are weighed.
        if (less && all.least < -80.f) all.least = -INFINITY;
        if (!greedy && !all.bad && (less || all.z > -INFINITY) && !(all.others < all.least - slack)) {           // (one call in a thousand)
            all.at = weigh<T>(v, logits, stats, splits, ranks, stop, less ? 2 : without >= 0 ? 1 : 0, all.ref, all.least, &far);
            all.z = all.at < V ? 0.f : -INFINITY;
        }
        // a draft was kept or turned down by less than its rows' sums are sure of (one in some ten thousand; asked here, where the loops' registers are free)
        if (unsettled) {
            unsettled = false;
            const int real = settle<T>(v, logits, stats, splits, ranks, doubt_at, &far);
            if (real != stop) {
                stop = real;
                cluster_all();                         // nobody reads what the next turn writes
                continue;
            }
        }
        // where nothing is left of p - q (or p is nothing but the draft), p itself
        if (!plain && !all.bad && all.z == -INFINITY && (less || without >= 0)) {
            plain = true;
            cluster_all();
            continue;
        }
        if (rank == 0 && threadIdx.x == 0) {
            const int s = blockIdx.x / ranks;
            accepted[s] = stop;
            next[s] = all.bad || all.z == -INFINITY ? -1 : all.at;
        }
        return;
    }
}

// 16 where the device can place a cluster of so many, otherwise 8
template <typename T>
int most_ranks() {
    static std::atomic<int> known[kMaxDevices] = {};
    std::atomic<int>& n = known[cmlb_device_index()];
    if (!n.load()) {
        int clusters = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(MOST_RANKS);
        cfg.blockDim = dim3(VT_THREADS);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = MOST_RANKS;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        const bool fits = cudaFuncSetAttribute(draft_token_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                          cudaOccupancyMaxActiveClusters(&clusters, draft_token_kernel<T>, &cfg) == cudaSuccess && clusters > 0;
        if (!fits) cudaGetLastError();
        n.store(fits ? MOST_RANKS : 8);
    }
    return n.load();
}

template <typename T>
int launch_verify(const Verify& v, const void* logits, int* accepted, int* next, void* work, cudaStream_t st) {
    const int drafts = v.d.rows - v.d.sequences, sides = v.d.logits ? 2 : 1;
    Stat* stats = static_cast<Stat*>(work);
    // parts of a row: 8 KB at least, all of them together about 8 CTAs an SM, or 4 for 16-bit rows, whose threads hold twice as many values (7 drafts of 4 sequences over 50,000 bf16 11.9 us, with 8 an SM
    // 13.4; 23 ragged sequences over 100,000 32.6 and 33.7, with 2 an SM 44; 32 sequences of 4 drafts over 128,000 fp32 41.5, with 16 an SM 41.4)
    int splits = 1;
    while (splits < VS_SPLITS && (long)drafts * sides * splits * 2 <= (sizeof(T) == 4 ? 8l : 4l) * cmlb_num_sms() && (size_t)v.vocab * sizeof(T) > (size_t)splits * 8192) splits *= 2;
    if (drafts)
        CMLB_CUDA(launch_chain(draft_stats_kernel<T>, dim3((unsigned)((long)drafts * sides * splits)), dim3(VS_THREADS), 0, 1, st, v, static_cast<const T*>(logits), sides, splits, stats));
    // as many CTAs a sequence as find an SM each, but 2,048 tokens at least
    const int most = most_ranks<T>();
    int ranks = 1;
    while (ranks < most && (long)v.d.sequences * ranks * 2 <= (ranks < 8 ? 2l * cmlb_num_sms() : cmlb_num_sms() / 2) && v.vocab > ranks * 2048) ranks *= 2;
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
    CMLB_REQUIRE(vocab > 0 && vocab <= MOST_VOCAB && ld >= vocab && (!d->logits || d->ld >= vocab), "%s: %d logits, strides %ld and %ld", who, vocab, ld, d->ld);
    CMLB_REQUIRE(d->tokens || d->rows == d->sequences, "%s: %d drafts without tokens", who, d->rows - d->sequences);
    CMLB_REQUIRE(d->random || d->temperature, "%s: no random numbers, and no temperatures that could do without", who);
    const uintptr_t words = (uintptr_t)d->first | (uintptr_t)d->tokens | (uintptr_t)d->temperature | (uintptr_t)d_accepted | (uintptr_t)d_next;
    CMLB_REQUIRE((((uintptr_t)d_logits | (uintptr_t)d->logits) & (dtype == CMLB200_DT_F32 ? 3 : 1)) == 0 && ((uintptr_t)d_work & 15) == 0 && ((uintptr_t)d->random & 7) == 0 && (words & 3) == 0,
                 "%s: pointers are not aligned to their types (workspace: 16 bytes)", who);
    const Verify v = {*d, ld, vocab};
    cudaStream_t st = as_stream(stream);
    if (dtype == CMLB200_DT_F32) return launch_verify<float>(v, d_logits, d_accepted, d_next, d_work, st);
    if (dtype == CMLB200_DT_BF16) return launch_verify<__nv_bfloat16>(v, d_logits, d_accepted, d_next, d_work, st);
    if (dtype == CMLB200_DT_F16) return launch_verify<__half>(v, d_logits, d_accepted, d_next, d_work, st);
    CMLB_REQUIRE(false, "%s: dtype %d", who, dtype);
    return CMLB200_EINVAL;
}
