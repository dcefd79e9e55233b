// Pages of paged caches: copies between pages in all pools at once, with the block table's entries following (a cache is compacted so),
// and forks, which share a sequence's full pages and copy the one that is still being filled.
//
// A page id names the same slot in every pool (a layer's keys, its values, their scales), and pools differ in the size of a page. One launch
// serves all of them: a CTA moves pieces of 16 KB of one page in one pool or four, four 16-byte loads a thread ahead of their stores, which keeps
// 96 KB of reads in flight on an SM (six CTAs of 40 registers a thread). Bound by memory: each byte is read once and written once. Measured: 900 pages of 16 layers (keys, values, scales; 946 MB read
// and written) in 158 us, 6.0 TB/s; four children of a sequence of 777 tokens in 32 layers in 3.0 us.
#include "lm_util.cuh"

namespace {

constexpr int PG_THREADS = 256, PG_LOADS = 4, PG_PIECE = PG_THREADS * PG_LOADS * 16;

template <typename V>
__device__ __forceinline__ void copy_piece(char* dst, const char* src, size_t bytes) {
    V* d = reinterpret_cast<V*>(dst);
    const V* s = reinterpret_cast<const V*>(src);
    const int n = (int)(bytes / sizeof(V));
    if constexpr (sizeof(V) == 16) {
        V v[PG_LOADS];
#pragma unroll
        for (int j = 0; j < PG_LOADS; j++) { const int i = j * PG_THREADS + threadIdx.x; if (i < n) v[j] = s[i]; }
#pragma unroll
        for (int j = 0; j < PG_LOADS; j++) { const int i = j * PG_THREADS + threadIdx.x; if (i < n) d[i] = v[j]; }
    } else {
        for (int i = threadIdx.x; i < n; i += PG_THREADS) d[i] = s[i];
    }
}
// piece `z` of the page `from` into `to`
__device__ __forceinline__ void copy_page(const cmlb200_page_pool& pool, int from, int to, int z) {
    const size_t at = (size_t)z * PG_PIECE;
    if (at >= pool.bytes) return;
    const size_t n = min(pool.bytes - at, (size_t)PG_PIECE);
    char* base = static_cast<char*>(pool.base);
    char* dst = base + (size_t)to * pool.stride + at;
    const char* src = base + (size_t)from * pool.stride + at;
    const uintptr_t all = (uintptr_t)base | pool.stride | pool.bytes;
    if ((all & 15) == 0) copy_piece<uint4>(dst, src, n);
    else if ((all & 3) == 0) copy_piece<uint32_t>(dst, src, n);
    else copy_piece<uint8_t>(dst, src, n);
}

// grid = (moves, ceil(pools / each) + (table ? 1 : 0), pieces of the largest page); a CTA takes `each` pools one after the other
__global__ void __launch_bounds__(PG_THREADS)
pages_copy_kernel(const cmlb200_pages p, const int2* __restrict__ moves, int n, int each) {
    dep_wait();
    dep_trigger();
    const int first = (int)blockIdx.y * each;
    if (first < p.pools) {
        const int2 m = moves[blockIdx.x];
        if ((unsigned)m.x < (unsigned)p.pages && (unsigned)m.y < (unsigned)p.pages && m.x != m.y)
            for (int k = first; k < min(first + each, p.pools); k++) copy_page(p.pool[k], m.x, m.y, blockIdx.z);
        return;
    }
    if (blockIdx.z) return;
    const size_t entries = (size_t)p.slots * p.table_ld;
    for (size_t i = (size_t)blockIdx.x * PG_THREADS + threadIdx.x; i < entries; i += (size_t)n * PG_THREADS) {
        const int id = p.table[i];
        int lo = 0, hi = n;                            // sources ascend: the first that is not below id
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (moves[mid].x < id) lo = mid + 1;
            else hi = mid;
        }
        if (lo < n && moves[lo].x == id && (unsigned)id < (unsigned)p.pages && (unsigned)moves[lo].y < (unsigned)p.pages) p.table[i] = moves[lo].y;
    }
}

// grid = (forks, pools + 1, pieces of the largest page); forks[i] = {parent slot, child slot, shared pages, the child's own next page or -1}
__global__ void __launch_bounds__(PG_THREADS)
pages_fork_kernel(const cmlb200_pages p, const int4* __restrict__ forks) {
    dep_wait();
    dep_trigger();
    const int4 f = forks[blockIdx.x];
    const bool own = f.w >= 0;
    if ((unsigned)f.x >= (unsigned)p.slots || (unsigned)f.y >= (unsigned)p.slots || f.x == f.y || f.z < 0 || f.z > p.table_ld - own || f.w >= p.pages) return;
    const int* from = p.table + (size_t)f.x * p.table_ld;
    if ((int)blockIdx.y < p.pools) {
        if (!own) return;
        const int page = from[f.z];
        if ((unsigned)page < (unsigned)p.pages && page != f.w) copy_page(p.pool[blockIdx.y], page, f.w, blockIdx.z);
        return;
    }
    int* to = p.table + (size_t)f.y * p.table_ld;
    for (int i = blockIdx.z * PG_THREADS + threadIdx.x; i < f.z + own; i += gridDim.z * PG_THREADS) to[i] = i < f.z ? from[i] : f.w;
}

int check_pages(const cmlb200_pages* p, const int* d_list, int n, const char* who) {
    CMLB_REQUIRE(p && d_list && n > 0, "%s: bad argument", who);
    CMLB_REQUIRE(p->pools >= 0 && p->pools < 65535 && (p->pools == 0 || p->pool) && p->pages > 0, "%s: %d pools of %d pages", who, p->pools, p->pages);
    CMLB_REQUIRE(p->most <= (size_t)65535 * PG_PIECE, "%s: pages of %zu bytes", who, p->most);
    CMLB_REQUIRE(!p->table || (p->slots > 0 && p->table_ld > 0), "%s: a block table of %d slots, %d entries each", who, p->slots, p->table_ld);
    return CMLB200_OK;
}
unsigned pieces_of(const cmlb200_pages* p) { return (unsigned)(p->most ? (p->most + PG_PIECE - 1) / PG_PIECE : 1); }

}  // namespace

extern "C" int cmlb200_pages_copy(const cmlb200_pages* p, const int* d_moves, int moves, void* stream) {
    static const char* who = "cmlb200_pages_copy";
    const int rc = check_pages(p, d_moves, moves, who);
    if (rc) return rc;
    CMLB_REQUIRE(((uintptr_t)d_moves & 7) == 0, "%s: the list of moves must be 8-byte aligned", who);
    CMLB_REQUIRE(p->pools > 0 || p->table, "%s: neither pools nor a table", who);
    // Four pools a CTA where CTAs would be many: pools of scales are little work for one (64 pools, 900 moves: 158 us, 168 by one pool a CTA; pages of a quarter: 109 and
    // 152), one where they are few (40 moves: 6.3 us, 9.7 by four).
    const int each = (long long)moves * p->pools >= 64LL * cmlb_num_sms() ? 4 : 1;
    CMLB_CUDA(launch_chain(pages_copy_kernel, dim3(moves, (p->pools + each - 1) / each + (p->table ? 1 : 0), pieces_of(p)), dim3(PG_THREADS), 0, 1, as_stream(stream), *p, (const int2*)d_moves,
                           moves, each));
    return CMLB200_OK;
}

extern "C" int cmlb200_pages_fork(const cmlb200_pages* p, const int* d_forks, int forks, void* stream) {
    static const char* who = "cmlb200_pages_fork";
    const int rc = check_pages(p, d_forks, forks, who);
    if (rc) return rc;
    CMLB_REQUIRE(p->table, "%s: no block table", who);
    CMLB_REQUIRE(((uintptr_t)d_forks & 15) == 0, "%s: the list of forks must be 16-byte aligned", who);
    CMLB_CUDA(launch_chain(pages_fork_kernel, dim3(forks, p->pools + 1, pieces_of(p)), dim3(PG_THREADS), 0, 1, as_stream(stream), *p, (const int4*)d_forks));
    return CMLB200_OK;
}
