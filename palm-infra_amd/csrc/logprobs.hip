// How likely tokens are: of rows of logits x [rows, V], for each row
//   log p_t = x_t - m - log S            the log probability of a given token t
//   H = log S - A / S                    the entropy, -sum p log p
// and the `top` likeliest tokens with their log probabilities, equal logits by their number, where
//   m = max x,   S = sum e^(x - m),   A = sum (x - m) e^(x - m),
// in one pass over the logits: a lane keeps m, S and A of what it has seen and rescales them when its m rises by d,
// S' = S e^-d, A' = (A - d S) e^-d.
//
// S is kept as the number of terms that are 1 (the largest, and equals) and the sum of the others: where the model is sure,
// log S is the small sum itself, which would drown in the rounding of 1 + it (p = 0.99996: 1 part in 1,000 of log p).
// Minus infinity is a token that cannot come (weight 0); a row without any other, with a NaN or with plus infinity has NaN as
// every result, as a softmax of it has.
//
// The likeliest: a wave keeps a list of candidates in LDS and the value that the last place of the list held when it was last
// put in order; a logit above it joins the list.  The first such value comes from the lanes' own maxima (at least `top`
// lanes hold one as large).  A candidate is a 64-bit number, the logit's bits in an order that integers have, then the
// token's number inverted: all differ, and the larger is the better one.
#include "common.h"

PALM_DEFINE_LAST_ERROR()

constexpr int LP_MOST = 64;                      // alternatives, at most
constexpr int LP_LIST = 128;                     // candidates a wave holds
constexpr int LP_PAD = 8;                        // of them read together
constexpr int LP_QUADS = 4;                      // reads of four logits a lane has on their way
constexpr int LP_TILE = WAVE * 4 * LP_QUADS;     // logits a wave takes at once
constexpr int LP_EACH = 4;                       // slices a lane of the wave that joins them has, at most
constexpr int LP_SLICES = LP_EACH * WAVE;        // slices of a row, at most
constexpr int LP_ROW_WAVES = 8;                  // waves of a block that has a row to itself
constexpr float LP_LOG2E = 1.4426950408889634f;

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));      // rows start where they may

struct Sums {
    float m, ones, s, a;                         // maximum; terms that are 1, the sum of the others, sum of t e^t
};

// 2^x as the one hardware instruction (results below 2^-126 come out as zero: they are added to a sum of at least 1)
__device__ inline float lp_exp(float t) { return __builtin_amdgcn_exp2f(t * LP_LOG2E); }

// What was seen against the maximum v.m, against `m`, which is no less.  (m is minus infinity where nothing was seen; NaN sums stay NaN.)
__device__ inline Sums moved_to(const Sums& v, float m) {
    if (v.m == m) return v;
    const float d = v.m - m, scale = lp_exp(d), all = v.ones + v.s;
    return Sums{m, 0.f, all * scale, scale == 0.f ? 0.f * v.a : (v.a + d * all) * scale};       // (d may be minus infinity)
}

// Over the wave, every lane's: rows of 16 lanes, then the rows' ends handed on, and the last lane has it.
template <int CTRL, int ROWS> __device__ inline float dpp(float old, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ inline float lanes_sum(float v) {
    v += dpp<0x111, 0xf>(0.f, v);                // row_shr 1, 2, 4, 8
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);                // row_bcast 15, 31
    v += dpp<0x143, 0xc>(0.f, v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), WAVE - 1));
}
__device__ inline float lanes_max(float v) {
    v = fmaxf(v, dpp<0x111, 0xf>(-INFINITY, v));
    v = fmaxf(v, dpp<0x112, 0xf>(-INFINITY, v));
    v = fmaxf(v, dpp<0x114, 0xf>(-INFINITY, v));
    v = fmaxf(v, dpp<0x118, 0xf>(-INFINITY, v));
    v = fmaxf(v, dpp<0x142, 0xa>(-INFINITY, v));
    v = fmaxf(v, dpp<0x143, 0xc>(-INFINITY, v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), WAVE - 1));
}
__device__ inline Sums of_wave(const Sums& v) {
    const float m = lanes_max(v.m);
    const Sums here = moved_to(v, m);
    return Sums{m, lanes_sum(here.ones), lanes_sum(here.s), lanes_sum(here.a)};
}

// a logit's place in the order of logits (both zeros are one)
__device__ inline int ordered(float x) {
    const int bits = __float_as_int(x + 0.0f);
    return bits ^ ((bits >> 31) & 0x7fffffff);
}
__device__ inline float unordered(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }
// (the sign bit turned: as unsigned numbers they are in order; no logit gives 0, which stands for no candidate)
__device__ inline uint64_t candidate(float logit, int token) { return (uint64_t)((uint32_t)ordered(logit) ^ 0x80000000u) << 32 | (uint32_t)~token; }
__device__ inline int token_of(uint64_t c) { return (int)~(uint32_t)c; }
__device__ inline float logit_of(uint64_t c) { return unordered((int)((uint32_t)(c >> 32) ^ 0x80000000u)); }

__device__ inline void wave_lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The first `n` candidates of the list, at most LP_LIST, become its best `keep` in order (zeros behind them where there are
// fewer).  Every candidate counts those that are better, eight read at a time.
template <int PER> __device__ inline void put_in_order_of(uint64_t* list, int n, int keep, int lane) {
    uint64_t mine[PER];
    int better[PER];
    if (lane < LP_PAD) list[n + lane] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        mine[i] = lane + i * WAVE < n ? list[lane + i * WAVE] : 0;
        better[i] = 0;
    }
    wave_lds_done();
    for (int c = 0; c < n; c += LP_PAD) {
        ulonglong2 two[LP_PAD / 2];
#pragma unroll
        for (int u = 0; u < LP_PAD / 2; ++u) two[u] = *reinterpret_cast<const ulonglong2*>(list + c + 2 * u);
#pragma unroll
        for (int u = 0; u < LP_PAD / 2; ++u)
#pragma unroll
            for (int i = 0; i < PER; ++i) better[i] += (two[u].x > mine[i] ? 1 : 0) + (two[u].y > mine[i] ? 1 : 0);
    }
    wave_lds_done();
    if (lane >= n && lane < keep) list[lane] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + i * WAVE < n && better[i] < keep) list[better[i]] = mine[i];
    wave_lds_done();
}
__device__ inline void put_in_order(uint64_t* list, int n, int keep, int lane) {
    wave_lds_done();
    if (n <= WAVE) put_in_order_of<1>(list, n, keep, lane);
    else put_in_order_of<LP_LIST / WAVE>(list, n, keep, lane);
}
// `candidates` of the lanes for which `joins` holds go behind the list's first `held`; returns how many there are then.
__device__ inline int append(uint64_t* list, int held, uint64_t who, bool joins, uint64_t candidate) {
    if (joins) list[held + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = candidate;
    return held + __popcll(who);
}

// A value that at least `count` lanes' `best` reach, the largest one or nearly (0: fewer lanes have one): bit by bit below what all lanes share, until
// just so many reach it.
__device__ inline uint32_t reached_by(uint32_t best, int count) {
    uint32_t reach = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t tried = reach | 1u << bit;
        const int n = __popcll(__ballot(best >= tried));
        if (n >= count) reach = tried;
        if (n == count) break;
    }
    return reach;
}

// Logits x[begin .. end) of a row: the lane's sums, and with TOP the wave's list of the best `top` in order.
template <bool TOP>
__device__ inline Sums scan(const float* __restrict__ x, int begin, int end, int top, uint64_t* list, int lane) {
    Sums mine = {-INFINITY, 0.f, 0.f, 0.f};
    int held = 0;                                // candidates in the list
    float joins_from = -INFINITY;                // the least logit that joins them
    float v[LP_QUADS][4], next[LP_QUADS][4];
    auto read = [&](int at, float (&to)[LP_QUADS][4]) {
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q) {
            const int p = at + q * WAVE * 4 + lane * 4;
            if (at + LP_TILE <= end) {           // the same in every lane
                const float4_any four = *reinterpret_cast<const float4_any*>(x + p);
#pragma unroll
                for (int e = 0; e < 4; ++e) to[q][e] = four[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) to[q][e] = p + e < end ? x[p + e] : -INFINITY;
            }
        }
    };
    if (begin < end) read(begin, v);
    for (int at = begin; at < end; at += LP_TILE) {
        if (at + LP_TILE < end) read(at + LP_TILE, next);
        float most = v[0][0];
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, v[q][e]);
        if (most > mine.m) mine = mine.m == -INFINITY ? Sums{most, 0.f, 0.f * mine.s, 0.f * mine.a} : moved_to(mine, most);     // (0 NaN: a NaN stays)
        const float from = mine.m == -INFINITY ? 0.f : mine.m;
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float t = v[q][e] - from, w = lp_exp(t);
                mine.ones += w == 1.f ? 1.f : 0.f;
                mine.s += w == 1.f ? 0.f : w;
                mine.a += w == 0.f ? 0.f : t * w;
            }
        if (TOP) {
            if (at == begin) {
                const uint32_t reach = reached_by((uint32_t)ordered(most) ^ 0x80000000u, top);
                joins_from = reach <= 0x007fffffu ? -INFINITY : unordered((int)(reach ^ 0x80000000u));     // (that is minus infinity's place)
            }
            if (__any(most >= joins_from)) {
                bool full = false;
#pragma unroll
                for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int token = at + q * WAVE * 4 + lane * 4 + e;
                        bool joins = v[q][e] >= joins_from && token < end;
                        uint64_t who = __ballot(joins);
                        if (who == 0) continue;
                        if (held + WAVE > LP_LIST) {     // (then more than `top`: what equals the last one may still come before it)
                            put_in_order(list, held, top, lane);
                            held = top;
                            full = true;
                            joins_from = fmaxf(joins_from, logit_of(list[top - 1]));
                            joins = v[q][e] >= joins_from && token < end;
                            who = __ballot(joins);
                        }
                        held = append(list, held, who, joins, candidate(v[q][e], token));
                    }
                if (full || held > LP_LIST / 2) {        // what comes from here on has a larger number: it has to be larger
                    put_in_order(list, held, top, lane);
                    held = min(held, top);
                    if (held == top) joins_from = fmaxf(joins_from, unordered(ordered(logit_of(list[top - 1])) + 1));     // (above infinity: a NaN, which nothing reaches)
                }
            }
        }
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = next[q][e];
    }
    if (TOP) put_in_order(list, held, top, lane);
    return mine;
}

// A given token's logit, asked for at the start.
struct Given {
    float logit;
    bool there;
    __device__ Given(const float* __restrict__ x, const int* __restrict__ tokens, int row, int V) {
        const int t = tokens ? tokens[row] : -1;
        there = t >= 0 && t < V;
        logit = x[there ? t : 0];
    }
};

// The row's results from its sums (in every lane) and its best candidates in order.
__device__ inline void finish(const Sums& all, const uint64_t* list, const Given& one, bool asked, int row, int top, float* __restrict__ given,
                              float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best, int lane) {
    const float more = all.s + (all.ones - 1.f), log_s = all.m == -INFINITY ? NAN : log1pf(more);
    if (lane == 0) {
        if (asked) given[row] = one.there ? (one.logit - all.m) - log_s : NAN;
        entropy[row] = log_s - all.a / (1.f + more);
    }
    if (lane < top) {
        const uint64_t c = list[lane];
        ids[(size_t)row * top + lane] = c ? token_of(c) : lane;            // (a row with a NaN may have fewer)
        best[(size_t)row * top + lane] = (logit_of(c) - all.m) - log_s;
    }
}

// Many rows: a block for each.
template <bool TOP>
__global__ __launch_bounds__(LP_ROW_WAVES * WAVE) void logprobs_row_kernel(const float* __restrict__ logits, int V, const int* __restrict__ tokens, int top,
                                                                         float* __restrict__ given, float* __restrict__ entropy, int* __restrict__ ids,
                                                                         float* __restrict__ best) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? LP_ROW_WAVES : 1][TOP ? LP_LIST + LP_PAD : 2];
    __shared__ Sums sums[LP_ROW_WAVES];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), row = blockIdx.x;
    const float* x = logits + (size_t)row * V;
    const Given one(x, tokens, row, V);
    const int per = (int)(((long long)V + LP_ROW_WAVES * LP_TILE - 1) / (LP_ROW_WAVES * LP_TILE)) * LP_TILE;
    const int begin = (int)min((long long)V, (long long)wave * per), end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = of_wave(scan<TOP>(x, begin, end, top, TOP ? lists[wave] : nullptr, lane));
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    if (wave != 0) return;
    const Sums all = of_wave(lane < LP_ROW_WAVES ? sums[lane] : Sums{-INFINITY, 0.f, 0.f, 0.f});
    if (TOP) {
        int held = top;
        for (int w = 1; w < LP_ROW_WAVES; ++w) {
            if (held + top > LP_LIST) { put_in_order(lists[0], held, top, lane); held = top; }
            if (lane < top) lists[0][held + lane] = lists[w][lane];
            held += top;
        }
        put_in_order(lists[0], held, top, lane);
    }
    finish(all, TOP ? lists[0] : nullptr, one, tokens != nullptr, row, top, given, entropy, ids, best, lane);
}

// Few rows: a wave for each slice of a row, whose sums and best candidates go to memory, ..
constexpr int LP_SLICE_WAVES = 4;
template <bool TOP>
__global__ __launch_bounds__(LP_SLICE_WAVES * WAVE) void logprobs_slice_kernel(const float* __restrict__ logits, int V, int per, int slices, int top,
                                                                              Sums* __restrict__ sums, uint64_t* __restrict__ found) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[LP_SLICE_WAVES][TOP ? LP_LIST + LP_PAD : 2];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int slice = blockIdx.x * LP_SLICE_WAVES + wave, row = blockIdx.y;
    if (slice >= slices) return;
    uint64_t* list = lists[wave];
    const int begin = slice * per, end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = of_wave(scan<TOP>(logits + (size_t)row * V, begin, end, top, list, lane));
    const size_t at = (size_t)row * slices + slice;
    if (lane == 0) sums[at] = mine;
    if (TOP && lane < top) found[at * top + lane] = list[lane];
}
// .. and a wave for each row that joins them, LP_EACH slices a lane.
template <bool TOP>
__global__ __launch_bounds__(WAVE) void logprobs_join_kernel(const float* __restrict__ logits, int V, int slices, const int* __restrict__ tokens, int top,
                                                             const Sums* __restrict__ sums, const uint64_t* __restrict__ found, float* __restrict__ given,
                                                             float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best) {
    __shared__ __attribute__((aligned(16))) uint64_t list[TOP ? LP_LIST + LP_PAD : 2];
    constexpr int AT_ONCE = 4;                           // candidates of a slice read together
    const int lane = threadIdx.x, row = blockIdx.x;
    const Given one(logits + (size_t)row * V, tokens, row, V);
    Sums each[LP_EACH];
    uint64_t ahead[LP_EACH][AT_ONCE];
    auto read = [&](int i0) {
#pragma unroll
        for (int k = 0; k < LP_EACH; ++k)
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int slice = lane + k * WAVE;
                ahead[k][u] = slice < slices && i0 + u < top ? found[((size_t)row * slices + slice) * top + i0 + u] : 0;
            }
    };
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < LP_EACH; ++k) {
        each[k] = lane + k * WAVE < slices ? sums[(size_t)row * slices + lane + k * WAVE] : Sums{-INFINITY, 0.f, 0.f, 0.f};
        m = fmaxf(m, each[k].m);
    }
    if (TOP) {
        read(0);
        // a slice's best stands first: what is to be taken reaches what the best of `top` lanes' slices reach (0: there are not so many)
        uint64_t first = ahead[0][0];
#pragma unroll
        for (int k = 1; k < LP_EACH; ++k) first = max(first, ahead[k][0]);
        uint64_t above = (uint64_t)reached_by((uint32_t)(first >> 32), top) << 32;
        above = above ? above - 1 : 0;
        int held = 0;
        bool more = true;
        for (int i0 = 0; i0 < top && more; i0 += AT_ONCE) {
            if (i0) read(i0);
            more = false;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                for (int k = 0; k < LP_EACH; ++k) {
                    bool joins = ahead[k][u] > above;
                    uint64_t who = __ballot(joins);
                    if (who == 0) continue;
                    if (held + WAVE > LP_LIST) {
                        put_in_order(list, held, top, lane);
                        held = top;
                        above = max(above, list[top - 1]);
                        joins = ahead[k][u] > above;
                        who = __ballot(joins);
                    }
                    held = append(list, held, who, joins, ahead[k][u]);
                    if (u == AT_ONCE - 1) more = true;   // (else what stands behind in every slice is smaller still)
                }
        }
        put_in_order(list, held, top, lane);
    }
    Sums all = {m, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < LP_EACH; ++k) {
        const Sums here = moved_to(each[k], m);
        all.ones += here.ones;
        all.s += here.s;
        all.a += here.a;
    }
    finish(of_wave(all), list, one, tokens != nullptr, row, top, given, entropy, ids, best, lane);
}

constexpr int LP_ROWS_APART = 256;               // rows from which each has a block of its own
constexpr int LP_WAVES_WANTED = 4096;            // below, slices are as short as it takes for so many waves

// Logits of a slice: whole tiles.
static int slice_size(int rows, int V) {
    const long long tiles = ((long long)V + LP_TILE - 1) / LP_TILE, all = tiles * rows;
    const long long least = (tiles + LP_SLICES - 1) / LP_SLICES, wanted = (all + LP_WAVES_WANTED - 1) / LP_WAVES_WANTED;
    return (int)((least > wanted ? least : wanted) * LP_TILE);
}
static int slices_of(int rows, int V) { return (int)(((long long)V + slice_size(rows, V) - 1) / slice_size(rows, V)); }

// Bytes of workspace, 0: none is needed.
PALM_API long long palm_token_logprobs_work(int rows, int V, int top) {
    if (rows <= 0 || V <= 0 || rows >= LP_ROWS_APART) return 0;
    return (long long)rows * slices_of(rows, V) * ((long long)sizeof(Sums) + 8ll * top);
}

// logits [rows, V] float32; tokens [rows] int32 or null; given [rows] (with tokens), entropy [rows], ids and best [rows, top].
PALM_API int palm_token_logprobs(hipStream_t stream, const float* logits, int rows, int V, const int* tokens, int top, void* work, long long work_bytes,
                                 float* given, float* entropy, int* ids, float* best) {
    PALM_CHECK(rows >= 0 && V > 0 && V <= 0x7fffffff - 64 * LP_TILE, "token_logprobs: %d rows of %d", rows, V);
    PALM_CHECK(top >= 0 && top <= LP_MOST && top <= V, "token_logprobs: the %d likeliest of %d tokens (%d at most)", top, V, LP_MOST);
    if (rows == 0) return 0;
    PALM_CHECK(work_bytes >= palm_token_logprobs_work(rows, V, top) && (work || work_bytes == 0), "token_logprobs: a workspace of %lld bytes is too small", work_bytes);
    if (rows >= LP_ROWS_APART) {
        if (top) logprobs_row_kernel<true><<<rows, LP_ROW_WAVES * WAVE, 0, stream>>>(logits, V, tokens, top, given, entropy, ids, best);
        else logprobs_row_kernel<false><<<rows, LP_ROW_WAVES * WAVE, 0, stream>>>(logits, V, tokens, top, given, entropy, ids, best);
        PALM_LAUNCHED();
        return 0;
    }
    const int per = slice_size(rows, V), slices = slices_of(rows, V);
    Sums* sums = (Sums*)work;
    uint64_t* found = (uint64_t*)(sums + (size_t)rows * slices);
    const dim3 grid((slices + LP_SLICE_WAVES - 1) / LP_SLICE_WAVES, rows);
    if (top) logprobs_slice_kernel<true><<<grid, LP_SLICE_WAVES * WAVE, 0, stream>>>(logits, V, per, slices, top, sums, found);
    else logprobs_slice_kernel<false><<<grid, LP_SLICE_WAVES * WAVE, 0, stream>>>(logits, V, per, slices, top, sums, found);
    PALM_LAUNCHED();
    if (top) logprobs_join_kernel<true><<<rows, WAVE, 0, stream>>>(logits, V, slices, tokens, top, sums, found, given, entropy, ids, best);
    else logprobs_join_kernel<false><<<rows, WAVE, 0, stream>>>(logits, V, slices, tokens, top, sums, found, given, entropy, ids, best);
    PALM_LAUNCHED();
    return 0;
}
