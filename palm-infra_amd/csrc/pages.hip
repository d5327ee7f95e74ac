// Pages of the cache copied to other pages, in every layer at once: what a branch of a sequence needs of the page that the
// sequence still writes, and how pages are moved together.  (The reference keeps one sequence in one flat buffer and has
// neither: engine/engine.h:34-63.)
//
// A storage is [layers, pages, bytes of a page]; a page is a number of runs of equal length, and a run's first
// tokens * token_bytes bytes are what its first `tokens` positions hold: keys [kv heads, 64, head size] are a run for each
// head, values, kept transposed [kv heads, head size, 64], one for each element of a head.  Only those bytes are read and
// written: positions behind stay as they were.
//
// What bounds it: every byte read once and written once for each copy.  A thread takes 16 bytes of a page and writes them to
// all copies of that page, so a page with many copies is read once.
#include "common.h"

#include <algorithm>
#include <new>
#include <vector>

PALM_DEFINE_LAST_ERROR()

constexpr int CP_THREADS = 256;
constexpr int CP_EACH = 4;               // chunks a thread has on their way together
constexpr int CP_GROUPS = 160;           // source pages of a launch, and copies: both go with its arguments
constexpr int CP_COPIES = 256;

struct Storage {
    char* base;
    long long layer_bytes, page_bytes;
    int runs, run_bytes, token_bytes;
};
struct CopyPlan {
    int src[CP_GROUPS], first[CP_GROUPS + 1], tokens[CP_GROUPS];       // copies first[i] .. first[i + 1] - 1 are of page src[i]
    int dst[CP_COPIES];
};

template <int BYTES> struct Chunk;
template <> struct Chunk<16> { using type = uint4; };
template <> struct Chunk<4> { using type = uint32_t; };
template <> struct Chunk<2> { using type = uint16_t; };

// The first `bytes` (even, fewer than all) of a chunk.
__device__ inline void store_first(char* to, uint4 v, int bytes) {
    if (bytes & 8) *reinterpret_cast<uint2*>(to) = make_uint2(v.x, v.y);
    const uint32_t word = bytes & 8 ? v.z : v.x, after = bytes & 8 ? v.w : v.y;
    if (bytes & 4) *reinterpret_cast<uint32_t*>(to + (bytes & 8)) = word;
    if (bytes & 2) *reinterpret_cast<uint16_t*>(to + (bytes & 12)) = (uint16_t)(bytes & 4 ? after : word);
}
__device__ inline void store_first(char* to, uint32_t v, int bytes) {
    if (bytes & 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)v;
}
__device__ inline void store_first(char*, uint16_t, int) {}

// grid (blocks of a page's chunks, source pages, layers * storages)
template <int BYTES>
__global__ __launch_bounds__(CP_THREADS) void copy_pages_kernel(Storage first, Storage second, int layers, CopyPlan plan) {
    using T = typename Chunk<BYTES>::type;
    const bool other = (int)blockIdx.z >= layers;
    const Storage s = other ? second : first;
    const int layer = (int)blockIdx.z - (other ? layers : 0), group = blockIdx.y;
    const int used = plan.tokens[group] * s.token_bytes;               // bytes of a run
    const unsigned per_run = (unsigned)(used + BYTES - 1) / BYTES, chunks = per_run * (unsigned)s.runs;
    const unsigned begin = blockIdx.x * (unsigned)(CP_THREADS * CP_EACH) + threadIdx.x;
    if (begin >= chunks) return;
    char* at = s.base + layer * s.layer_bytes;
    const char* from = at + plan.src[group] * s.page_bytes;
    T held[CP_EACH];
    long long place[CP_EACH];
    int rest[CP_EACH];                                                 // bytes from the chunk's start to the end of what is used; 0: no chunk
#pragma unroll
    for (int i = 0; i < CP_EACH; ++i) {
        const unsigned c = begin + i * CP_THREADS;
        rest[i] = 0;
        if (c < chunks) {
            const unsigned run = c / per_run, in_run = c % per_run * BYTES;
            place[i] = (long long)run * s.run_bytes + in_run;
            rest[i] = used - (int)in_run;
            held[i] = *reinterpret_cast<const T*>(from + place[i]);    // (a run is whole chunks long)
        }
    }
    for (int d = plan.first[group]; d < plan.first[group + 1]; ++d) {
        char* to = at + plan.dst[d] * s.page_bytes;
#pragma unroll
        for (int i = 0; i < CP_EACH; ++i) {
            if (rest[i] >= BYTES) {
                *reinterpret_cast<T*>(to + place[i]) = held[i];
            } else if (rest[i] > 0) {                                  // the last positions' chunk: its halves, quarters and eighths as they are used
                store_first(to + place[i], held[i], rest[i]);
            }
        }
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
            if (groups == 0 || plan.src[groups - 1] != src[i] || plan.tokens[groups - 1] != held(i)) {
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
            chunks = std::max(chunks, (long long)s->runs * ((most * s->token_bytes + bytes - 1) / bytes));
        }
        const long long blocks = (chunks + CP_THREADS * CP_EACH - 1) / (CP_THREADS * CP_EACH);
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
        PALM_CHECK(s->runs > 0 && s->token_bytes > 0 && (long long)s->token_bytes * page_tokens == s->run_bytes && s->run_bytes % 2 == 0,
                   "copy_pages: %d runs of %d bytes, %d a position", s->runs, s->run_bytes, s->token_bytes);
    }
    if (n == 0 || layers == 0) return 0;
    try {
        return launch_copies(stream, a, b, n_storages, layers, pages, page_tokens, src, dst, tokens, n);
    } catch (const std::bad_alloc&) {
        return palm_fail("copy_pages: no host memory for %d copies", n);
    }
}
