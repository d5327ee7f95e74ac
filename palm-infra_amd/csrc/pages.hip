// Pages of the cache copied to other pages, in every layer at once: what a branch of a sequence needs of the page that the
// sequence still writes, and how pages are moved together.  (The reference keeps one sequence in one flat buffer and has
// neither: engine/engine.h:34-63.)
//
// A storage is [layers, pages, bytes of a page]; a page is a number of runs of equal length, and a run's first
// tokens * token_bytes bytes are what its first `tokens` positions hold: keys [kv heads, 64, head size] are a run for each
// head, values, kept transposed [kv heads, head size, 64], one for each element of a head.  Positions behind those stay as they were.
//
// What bounds it: every byte read once and written once for each copy.  A thread takes 16 bytes of a page and writes them to
// two copies of that page.  120 pages of 36 layers (2.26 GB read and written) 363 us, 6.2 TB/s; four chunks
// a thread 417, blocks of 512 threads 388; a copy of one page's 37 positions 5 us.
#include "common.h"

#include <algorithm>
#include <new>
#include <vector>

PALM_DEFINE_LAST_ERROR()

constexpr int CP_THREADS = 256;
constexpr int CP_GROUPS = 160;           // source pages of a launch, and copies: both go with its arguments
constexpr int CP_COPIES = 256;
// Copies that a thread writes of what it has read; a page with more is read again by others, from the caches.  us, eight to each of six pages, sixteen to each of three:
// all of them 106 77, four at once 106 72, two 93 67, one 108 68.
constexpr int CP_AT_ONCE = 2;

struct Storage {
    char* base;
    long long layer_bytes, page_bytes;
    int runs, run_bytes, token_bytes;
};
struct CopyPlan {
    int src[CP_GROUPS], first[CP_GROUPS + 1], tokens[CP_GROUPS];       // copies first[i] .. first[i + 1] - 1 are of page src[i], CP_AT_ONCE at most
    int dst[CP_COPIES];
};

// Bytes from a run's start that a copy writes, where it uses `used`: whole lines of memory, what is not used with what it held.  A line written in
// part costs memory a read of it and a write all the same, and waits for both: six pages of 4 to 58 positions to eight others each, in
// 36 layers of 8 heads of 128, 149 us with the bytes that are used alone and 122 with whole lines (half of the values' lines are written in part).
constexpr int CP_LINE = 128;
__host__ __device__ inline int touched_bytes(int used, int run_bytes) { return min(run_bytes, (used + CP_LINE - 1) / CP_LINE * CP_LINE); }

// What is written is not read again soon, nor what it replaces: marked so, both leave the caches to what is read (120 whole pages 374 us without, 370 with it, the
// six pages above 122 without, 117 with the writes marked, 106 with the reads of what they replace, 93 by two copies a thread).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ inline void store_past(char* p, uint4 v) { __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(p)); }
__device__ inline void store_past(char* p, uint32_t v) { __builtin_nontemporal_store(v, reinterpret_cast<uint32_t*>(p)); }
__device__ inline void store_past(char* p, uint16_t v) { __builtin_nontemporal_store(v, reinterpret_cast<uint16_t*>(p)); }
__device__ inline uint4 load_past(const uint4* p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ inline uint32_t load_past(const uint32_t* p) { return __builtin_nontemporal_load(p); }
__device__ inline uint16_t load_past(const uint16_t* p) { return __builtin_nontemporal_load(p); }

template <int BYTES> struct Chunk;
template <> struct Chunk<16> { using type = uint4; };
template <> struct Chunk<4> { using type = uint32_t; };
template <> struct Chunk<2> { using type = uint16_t; };

// `v` with what it has beyond its first `bytes` (even) bytes taken from `old`.
__device__ inline uint32_t first_of(uint32_t v, uint32_t old, int bytes) { return bytes >= 4 ? v : bytes == 2 ? (v & 0xffffu) | (old & 0xffff0000u) : old; }
__device__ inline uint4 first_of(uint4 v, uint4 old, int bytes) {
    return make_uint4(first_of(v.x, old.x, bytes), first_of(v.y, old.y, max(0, bytes - 4)), first_of(v.z, old.z, max(0, bytes - 8)),
                      first_of(v.w, old.w, max(0, bytes - 12)));
}
__device__ inline uint16_t first_of(uint16_t v, uint16_t old, int bytes) { return bytes >= 2 ? v : old; }

// grid (blocks of a page's chunks, source pages, layers * storages); a thread has one chunk.
template <int BYTES>
__global__ __launch_bounds__(CP_THREADS) void copy_pages_kernel(Storage first, Storage second, int layers, CopyPlan plan) {
    using T = typename Chunk<BYTES>::type;
    const bool other = (int)blockIdx.z >= layers;
    const Storage s = other ? second : first;
    const int layer = (int)blockIdx.z - (other ? layers : 0), group = blockIdx.y;
    const int used = plan.tokens[group] * s.token_bytes, touched = touched_bytes(used, s.run_bytes);     // bytes of a run
    const unsigned per_run = (unsigned)(touched + BYTES - 1) / BYTES, chunk = blockIdx.x * (unsigned)CP_THREADS + threadIdx.x;
    if (chunk >= per_run * (unsigned)s.runs) return;
    const unsigned run = chunk / per_run, in_run = chunk % per_run * BYTES;
    char* at = s.base + layer * s.layer_bytes + (long long)run * s.run_bytes + in_run;
    const int rest = used - (int)in_run;                               // bytes from the chunk's start to the end of what is used
    const int d0 = plan.first[group], d1 = plan.first[group + 1];
    const T* from = reinterpret_cast<const T*>(at + plan.src[group] * s.page_bytes);       // (a run is whole chunks long)
    // (a page that is copied once is not read again: 120 whole pages 370 us without that, 363 with it)
    const T held = d1 - d0 == 1 ? load_past(from) : *from;
    if (__any(rest < BYTES)) {
        T old;                                                         // what the next copy's page holds there
        if (rest < BYTES) old = load_past(reinterpret_cast<const T*>(at + plan.dst[d0] * s.page_bytes));
        for (int d = d0; d < d1; ++d) {
            const T now = rest < BYTES ? first_of(held, old, max(0, rest)) : held;
            if (d + 1 < d1 && rest < BYTES) old = load_past(reinterpret_cast<const T*>(at + plan.dst[d + 1] * s.page_bytes));
            store_past(at + plan.dst[d] * s.page_bytes, now);
        }
    } else {
        for (int d = d0; d < d1; ++d) store_past(at + plan.dst[d] * s.page_bytes, held);
    }
}

static int launch_copies(hipStream_t stream, const Storage& a, const Storage& b, int n_storages, int layers, int pages, int page_tokens,
                         const int* src, const int* dst, const int* tokens, int n) {
    std::vector<unsigned char> mark(pages, 0);                         // 1: read, 2: written
    for (int i = 0; i < n; ++i) {
        PALM_CHECK(src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages, "copy_pages: copy %d goes from page %d to %d of %d", i, src[i], dst[i], pages);
        PALM_CHECK(!tokens || (tokens[i] >= 0 && tokens[i] <= page_tokens), "copy_pages: copy %d has %d of %d positions", i, tokens ? tokens[i] : 0, page_tokens);
        PALM_CHECK(!(mark[dst[i]] & 2), "copy_pages: page %d is written twice", dst[i]);
        mark[dst[i]] |= 2;
        mark[src[i]] |= 1;
    }
    for (int i = 0; i < n; ++i) PALM_CHECK(!(mark[dst[i]] & 1), "copy_pages: page %d is both read and written", dst[i]);
    if (a.page_bytes == 0 && (n_storages < 2 || b.page_bytes == 0)) return 0;       // (a state of no elements: nothing to copy)
    std::vector<int> order(n);
    for (int i = 0; i < n; ++i) order[i] = i;
    auto held = [&](int i) { return tokens ? tokens[i] : page_tokens; };
    std::sort(order.begin(), order.end(), [&](int x, int y) {
        return src[x] != src[y] ? src[x] < src[y] : held(x) != held(y) ? held(x) < held(y) : x < y;
    });
    int bytes = 16;
    for (const Storage* s : {&a, &b}) {
        if (s == &b && n_storages < 2) break;
        while ((reinterpret_cast<uintptr_t>(s->base) | s->page_bytes | s->run_bytes) % bytes) bytes = bytes == 16 ? 4 : 2;
    }
    int done = 0;
    while (done < n) {
        CopyPlan plan;
        int groups = 0, copies = 0, most = 0;
        for (; done < n && copies < CP_COPIES; ++done) {
            const int i = order[done];
            if (held(i) == 0) continue;
            if (groups == 0 || plan.src[groups - 1] != src[i] || plan.tokens[groups - 1] != held(i) || copies - plan.first[groups - 1] == CP_AT_ONCE) {
                if (groups == CP_GROUPS) break;
                plan.src[groups] = src[i];
                plan.tokens[groups] = held(i);
                plan.first[groups++] = copies;
                most = std::max(most, held(i));
            }
            plan.dst[copies++] = dst[i];
            plan.first[groups] = copies;
        }
        if (groups == 0) break;
        long long chunks = 0;
        for (const Storage* s : {&a, &b}) {
            if (s == &b && n_storages < 2) break;
            chunks = std::max(chunks, (long long)s->runs * ((touched_bytes(most * s->token_bytes, s->run_bytes) + bytes - 1) / bytes));
        }
        const long long blocks = (chunks + CP_THREADS - 1) / CP_THREADS;
        PALM_CHECK(chunks < 1ll << 31 && layers * n_storages <= 65535, "copy_pages: %d layers of pages of %lld bytes are more than one launch takes", layers, a.page_bytes);
        const dim3 grid((unsigned)blocks, groups, layers * n_storages);
        if (bytes == 16) copy_pages_kernel<16><<<grid, CP_THREADS, 0, stream>>>(a, b, layers, plan);
        else if (bytes == 4) copy_pages_kernel<4><<<grid, CP_THREADS, 0, stream>>>(a, b, layers, plan);
        else copy_pages_kernel<2><<<grid, CP_THREADS, 0, stream>>>(a, b, layers, plan);
        PALM_LAUNCHED();
    }
    return 0;
}

// One storage or two (keys and values) of `layers` times `pages` pages of page_tokens positions.  src, dst, tokens: in host memory; tokens may be
// null (all positions).  Refused: a page that does not exist, one written twice, one both read and written.
PALM_API int palm_copy_pages(hipStream_t stream, void* base0, int runs0, int run_bytes0, int token_bytes0, void* base1, int runs1, int run_bytes1,
                             int token_bytes1, int layers, int pages, int page_tokens, const int* src, const int* dst, const int* tokens, int n) {
    PALM_CHECK(n >= 0 && layers >= 0 && pages >= 0 && page_tokens > 0, "copy_pages: copies=%d layers=%d pages=%d", n, layers, pages);
    auto storage = [&](void* base, int runs, int run_bytes, int token_bytes) {
        const long long page = (long long)runs * run_bytes;
        return Storage{(char*)base, page * pages, page, runs, run_bytes, token_bytes};
    };
    const Storage a = storage(base0, runs0, run_bytes0, token_bytes0), b = storage(base1, runs1, run_bytes1, token_bytes1);
    const int n_storages = base1 ? 2 : 1;
    for (const Storage* s : {&a, &b}) {
        if (s == &b && n_storages < 2) break;
        PALM_CHECK(s->runs > 0 && s->token_bytes >= 0 && (long long)s->token_bytes * page_tokens == s->run_bytes && s->run_bytes % 2 == 0,
                   "copy_pages: %d runs of %d bytes, %d a position", s->runs, s->run_bytes, s->token_bytes);
    }
    if (n == 0 || layers == 0) return 0;
    try {
        return launch_copies(stream, a, b, n_storages, layers, pages, page_tokens, src, dst, tokens, n);
    } catch (const std::bad_alloc&) {
        return palm_fail("copy_pages: no host memory for %d copies", n);
    }
}
