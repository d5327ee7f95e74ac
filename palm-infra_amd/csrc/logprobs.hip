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
constexpr int LP_SLICES = 64;                    // slices of a row, at most: one a lane of the wave that joins them
constexpr int LP_LIST = 256;                     // candidates a wave holds
constexpr int LP_QUADS = 4;                      // reads of four logits a lane has on their way
constexpr int LP_TILE = WAVE * 4 * LP_QUADS;     // logits a wave takes at once
constexpr int LP_ROW_WAVES = 8;                  // waves of a block that has a row to itself
constexpr float LP_LOG2E = 1.4426950408889634f;

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));      // rows start where they may

struct Sums {
    float m, ones, s, a;                         // maximum; terms that are 1, the sum of the others, sum of t e^t
};

// 2^x as the one hardware instruction (results below 2^-126 come out as zero: they are added to a sum of at least 1)
__device__ inline float lp_exp(float t) { return __builtin_amdgcn_exp2f(t * LP_LOG2E); }

// What b has seen joins a.  (m is minus infinity where nothing was seen; NaN sums stay NaN.)
__device__ inline void join(Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), from = m == -INFINITY ? 0.f : m;
    auto moved = [&](const Sums& x, float& ones, float& s, float& t) {
        if (x.m == m) { ones = x.ones; s = x.s; t = x.a; return; }
        const float d = x.m == -INFINITY ? 0.f : x.m - from, scale = x.m == -INFINITY ? 0.f : lp_exp(d), all = x.ones + x.s;
        ones = 0.f;
        s = all * scale;
        t = scale == 0.f ? 0.f * x.a : (x.a + d * all) * scale;        // (d may be minus infinity then)
    };
    float o0, s0, t0, o1, s1, t1;
    moved(a, o0, s0, t0);
    moved(b, o1, s1, t1);
    a = Sums{m, o0 + o1, s0 + s1, t0 + t1};
}
__device__ inline Sums of_wave(Sums v) {
#pragma unroll
    for (int off = WAVE / 2; off > 0; off >>= 1) {
        const Sums other = {__shfl_xor(v.m, off, WAVE), __shfl_xor(v.ones, off, WAVE), __shfl_xor(v.s, off, WAVE), __shfl_xor(v.a, off, WAVE)};
        join(v, other);
    }
    return v;
}

// a logit's place in the order of logits (both zeros are one)
__device__ inline int ordered(float x) {
    const int bits = __float_as_int(x + 0.0f);
    return bits ^ ((bits >> 31) & 0x7fffffff);
}
__device__ inline float unordered(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }
// (the sign bit turned: as unsigned numbers they are in order; no logit gives 0, which stands for no candidate)
__device__ inline uint64_t candidate(int order, int token) { return (uint64_t)((uint32_t)order ^ 0x80000000u) << 32 | (uint32_t)~token; }
__device__ inline int token_of(uint64_t c) { return (int)~(uint32_t)c; }
__device__ inline float logit_of(uint64_t c) { return unordered((int)((uint32_t)(c >> 32) ^ 0x80000000u)); }

__device__ inline void wave_lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The first `n` candidates of the list, at most LP_LIST, become its best `keep` in order (zeros behind them where there are
// fewer).  Every candidate counts those that are better.
__device__ inline void put_in_order(uint64_t* list, int n, int keep, int lane) {
    wave_lds_done();
    uint64_t mine[LP_LIST / WAVE];
    int better[LP_LIST / WAVE];
#pragma unroll
    for (int i = 0; i < LP_LIST / WAVE; ++i) {
        mine[i] = lane + i * WAVE < n ? list[lane + i * WAVE] : 0;
        better[i] = 0;
    }
    for (int c = 0; c < n; ++c) {
        const uint64_t other = list[c];
#pragma unroll
        for (int i = 0; i < LP_LIST / WAVE; ++i) better[i] += other > mine[i] ? 1 : 0;
    }
    wave_lds_done();
    if (lane >= n && lane < keep) list[lane] = 0;
#pragma unroll
    for (int i = 0; i < LP_LIST / WAVE; ++i)
        if (lane + i * WAVE < n && better[i] < keep) list[better[i]] = mine[i];
    wave_lds_done();
}

// Logits x[begin .. end) of a row: the lane's sums, and with TOP the wave's list of the best `top` in order.
template <bool TOP>
__device__ inline Sums scan(const float* __restrict__ x, int begin, int end, int top, uint64_t* list, int lane) {
    Sums mine = {-INFINITY, 0.f, 0.f, 0.f};
    int held = 0, above = (int)0x80000000;       // candidates in the list; what a logit has to be above to join
    bool first = true;
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
        if (most > mine.m) {
            const float d = mine.m == -INFINITY ? 0.f : mine.m - most, scale = mine.m == -INFINITY ? 0.f : lp_exp(d), all = mine.ones + mine.s;
            mine = Sums{most, 0.f, all * scale, scale == 0.f ? 0.f * mine.a : (mine.a + d * all) * scale};
        }
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
            int best = ordered(v[0][0]);
#pragma unroll
            for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) best = max(best, ordered(v[q][e]));
            if (first) {
                // the largest value that `top` lanes' maxima reach, bit by bit
                first = false;
                uint32_t reach = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t tried = reach | 1u << bit;
                    if (__popcll(__ballot(((uint32_t)best ^ 0x80000000u) >= tried)) >= top) reach = tried;
                }
                above = reach == 0 ? (int)0x80000000 : (int)((reach - 1) ^ 0x80000000u);
            }
            if (__any(best > above)) {
                for (int j = 0; j < LP_QUADS * 4; ++j) {
                    float value = v[0][0];
#pragma unroll
                    for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) value = j == q * 4 + e ? v[q][e] : value;
                    const int token = at + j / 4 * WAVE * 4 + lane * 4 + j % 4, o = ordered(value);
                    const bool joins = o > above && token < end;
                    const uint64_t who = __ballot(joins);
                    if (who == 0) continue;
                    if (held + WAVE > LP_LIST) {         // (then more than `top`: what equals the last one may still come before it)
                        put_in_order(list, held, top, lane);
                        held = top;
                        above = max(above, ordered(logit_of(list[top - 1])) - 1);
                    }
                    if (joins) list[held + __popcll(who & ((1ull << lane) - 1))] = candidate(o, token);
                    held += __popcll(who);
                }
                if (held >= top) {                       // what comes from here on has a larger number: it has to be larger
                    put_in_order(list, held, top, lane);
                    held = top;
                    above = max(above, ordered(logit_of(list[top - 1])));
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

// The row's results from its sums (in every lane) and its best candidates in order.
__device__ inline void finish(const Sums& all, const uint64_t* list, const float* __restrict__ x, const int* __restrict__ tokens, int row, int V, int top,
                              float* __restrict__ given, float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best, int lane) {
    const float more = all.s + (all.ones - 1.f), log_s = all.m == -INFINITY ? NAN : log1pf(more);
    if (lane == 0) {
        if (tokens) {
            const int t = tokens[row];
            given[row] = t >= 0 && t < V ? (x[t] - all.m) - log_s : NAN;
        }
        entropy[row] = log_s - all.a / (1.f + more);
    }
    if (lane < top) {
        const uint64_t c = list[lane];
        ids[(size_t)row * top + lane] = token_of(c);
        best[(size_t)row * top + lane] = (logit_of(c) - all.m) - log_s;
    }
}

// Many rows: a block for each.
template <bool TOP>
__global__ __launch_bounds__(LP_ROW_WAVES * WAVE) void logprobs_row_kernel(const float* __restrict__ logits, int V, const int* __restrict__ tokens, int top,
                                                                         float* __restrict__ given, float* __restrict__ entropy, int* __restrict__ ids,
                                                                         float* __restrict__ best) {
    __shared__ uint64_t lists[TOP ? LP_ROW_WAVES : 1][TOP ? LP_LIST : 1];
    __shared__ Sums sums[LP_ROW_WAVES];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), row = blockIdx.x;
    const float* x = logits + (size_t)row * V;
    const int per = (int)(((long long)V + LP_ROW_WAVES * LP_TILE - 1) / (LP_ROW_WAVES * LP_TILE)) * LP_TILE;
    const int begin = (int)min((long long)V, (long long)wave * per), end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = of_wave(scan<TOP>(x, begin, end, top, TOP ? lists[wave] : nullptr, lane));
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    if (wave != 0) return;
    Sums all = sums[0];
    for (int w = 1; w < LP_ROW_WAVES; ++w) join(all, sums[w]);
    if (TOP) {
        int held = top;
        for (int w = 1; w < LP_ROW_WAVES; ++w) {
            if (held + top > LP_LIST) { put_in_order(lists[0], held, top, lane); held = top; }
            if (lane < top) lists[0][held + lane] = lists[w][lane];
            held += top;
        }
        put_in_order(lists[0], held, top, lane);
    }
    finish(all, TOP ? lists[0] : nullptr, x, tokens, row, V, top, given, entropy, ids, best, lane);
}

// Few rows: a wave for each slice of a row, whose sums and best candidates go to memory, ..
template <bool TOP>
__global__ __launch_bounds__(WAVE) void logprobs_slice_kernel(const float* __restrict__ logits, int V, int per, int top, Sums* __restrict__ sums,
                                                              uint64_t* __restrict__ found) {
    __shared__ uint64_t list[TOP ? LP_LIST : 1];
    const int lane = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
    const int begin = slice * per, end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = of_wave(scan<TOP>(logits + (size_t)row * V, begin, end, top, list, lane));
    const size_t at = (size_t)row * gridDim.x + slice;
    if (lane == 0) sums[at] = mine;
    if (TOP && lane < top) found[at * top + lane] = list[lane];
}
// .. and a wave for each row that joins them.
template <bool TOP>
__global__ __launch_bounds__(WAVE) void logprobs_join_kernel(const float* __restrict__ logits, int V, int slices, const int* __restrict__ tokens, int top,
                                                             const Sums* __restrict__ sums, const uint64_t* __restrict__ found, float* __restrict__ given,
                                                             float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best) {
    __shared__ uint64_t list[TOP ? LP_LIST : 1];
    const int lane = threadIdx.x, row = blockIdx.x;
    const Sums none = {-INFINITY, 0.f, 0.f, 0.f};
    const Sums all = of_wave(lane < slices ? sums[(size_t)row * slices + lane] : none);
    if (TOP) {
        const uint64_t* mine = found + ((size_t)row * slices + min(lane, slices - 1)) * top;
        // a slice's best stands first: the list takes what reaches the best that `top` slices have, some at a time
        int held = 0;
        uint64_t above = 0;
        for (int i = 0; i < top; ++i) {
            const uint64_t c = lane < slices ? mine[i] : 0;
            const bool joins = c > above;
            const uint64_t who = __ballot(joins);
            if (who == 0) break;
            if (held + WAVE > LP_LIST) {
                put_in_order(list, held, top, lane);
                held = top;
                above = list[top - 1];
            }
            if (joins) list[held + __popcll(who & ((1ull << lane) - 1))] = c;
            held += __popcll(who);
        }
        put_in_order(list, held, top, lane);
    }
    finish(all, list, logits + (size_t)row * V, tokens, row, V, top, given, entropy, ids, best, lane);
}

static int slice_size(int V) { return (int)(((long long)V + (long long)LP_SLICES * 4 * WAVE - 1) / ((long long)LP_SLICES * 4 * WAVE)) * 4 * WAVE; }
static int slices_of(int V) { return (V + slice_size(V) - 1) / slice_size(V); }
constexpr int LP_ROWS_APART = 256;               // rows from which each has a block of its own

// Bytes of workspace, 0: none is needed.
PALM_API long long palm_token_logprobs_work(int rows, int V, int top) {
    if (rows <= 0 || V <= 0 || rows >= LP_ROWS_APART) return 0;
    return (long long)rows * slices_of(V) * ((long long)sizeof(Sums) + 8ll * top);
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
    const int per = slice_size(V), slices = slices_of(V);
    Sums* sums = (Sums*)work;
    uint64_t* found = (uint64_t*)(sums + (size_t)rows * slices);
    const dim3 grid(slices, rows);
    if (top) logprobs_slice_kernel<true><<<grid, WAVE, 0, stream>>>(logits, V, per, top, sums, found);
    else logprobs_slice_kernel<false><<<grid, WAVE, 0, stream>>>(logits, V, per, top, sums, found);
    PALM_LAUNCHED();
    if (top) logprobs_join_kernel<true><<<rows, WAVE, 0, stream>>>(logits, V, slices, tokens, top, sums, found, given, entropy, ids, best);
    else logprobs_join_kernel<false><<<rows, WAVE, 0, stream>>>(logits, V, slices, tokens, top, sums, found, given, entropy, ids, best);
    PALM_LAUNCHED();
    return 0;
}
