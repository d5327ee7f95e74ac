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
// The likeliest: the largest of every 16 logits (a lane's of a tile; more of them in rows of more than 262,144) are kept beside the pass.  What a
// share of `top` of the threads of every wave of a block find among theirs is reached by as many logits at least and by not many more: only
// where a group's largest reaches it are logits looked at again.  A candidate is a 64-bit number, the logit's bits in an order that integers have, then the
// token's number inverted: all differ, and the larger is the better one.  A list of candidates in LDS is put in order by every one's count of those that
// are better.  Where too many logits are equal for that (masks that leave few tokens), a block goes over the row once more, its waves with a list each.
#include "common.h"

PALM_DEFINE_LAST_ERROR()

constexpr int LP_MOST = 64;                      // alternatives, at most
constexpr int LP_LIST = 256;                     // candidates a wave holds
constexpr int LP_PAD = 8;                        // of them read together
constexpr int LP_QUADS = 4;                      // reads of four logits a lane has on their way
constexpr int LP_TILE = WAVE * 4 * LP_QUADS;     // logits a wave takes at once
constexpr int LP_EACH = 4;                       // slices a lane of the wave that joins them has, at most
constexpr int LP_SLICES = LP_EACH * WAVE;        // slices of a row, at most
constexpr int LP_ROW_WAVES = 8;                  // waves of a block that has a row to itself
constexpr int LP_GROUPS = 16384;                 // groups of a row, at most
constexpr int LP_CHOSEN = 512;                   // groups that are looked at again, at most
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
    else if (n <= 2 * WAVE) put_in_order_of<2>(list, n, keep, lane);
    else put_in_order_of<LP_LIST / WAVE>(list, n, keep, lane);
}
// `candidates` of the lanes for which `joins` holds go behind the list's first `held`; returns how many there are then.
__device__ inline int append(uint64_t* list, int held, uint64_t who, bool joins, uint64_t candidate) {
    if (joins) list[held + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = candidate;
    return held + __popcll(who);
}

// LP_TILE logits from `at` on, a lane's four by four; beyond `end` minus infinity.  They pass once, marked so: 2,047 rows of 151,936 183 us, 6.8 TB/s (208 without),
// 400 rows 40.5 (45.3), 512 with 20 alternatives 57.8 (63.8), 100 of 50,000 with five 14.1 (15.0); 300 of 50,000, which the cache beside the memory held, 15.8 (14.4).
template <int QUADS> __device__ inline void read_tile(const float* __restrict__ x, int at, int end, int lane, float (&to)[QUADS][4]) {
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
        const int p = at + q * WAVE * 4 + lane * 4;
        if (at + QUADS * WAVE * 4 <= end) {      // the same in every lane
            const float4_any four = __builtin_nontemporal_load(reinterpret_cast<const float4_any*>(x + p));
#pragma unroll
            for (int e = 0; e < 4; ++e) to[q][e] = four[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) to[q][e] = p + e < end ? x[p + e] : -INFINITY;
        }
    }
}

// Logits x[begin .. end) of a row, begin on a group's border: the wave's sums, and with TOP the groups' largest (a lane's of `span` tiles).
template <bool TOP>
__device__ inline Sums scan(const float* __restrict__ x, int begin, int end, int span, float* largest, int lane) {
    float m = -INFINITY, ones = 0.f, sum = 0.f, a = 0.f;       // the wave's maximum so far; against it the lane's own sums
    float v[LP_QUADS][4], next[LP_QUADS][4], of_group = -INFINITY;
    if (begin < end) read_tile<LP_QUADS>(x, begin, end, lane, v);
    int tile = begin / LP_TILE;
    for (int at = begin; at < end; at += LP_TILE, ++tile) {
        if (at + LP_TILE < end) read_tile<LP_QUADS>(x, at + LP_TILE, end, lane, next);
        float most = v[0][0];
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, v[q][e]);
        if (TOP) {
            of_group = fmaxf(of_group, most);
            if (span == 1 || (tile + 1) % span == 0 || at + LP_TILE >= end) {
                largest[tile / span * WAVE + lane] = of_group;
                of_group = -INFINITY;
            }
        }
        if (__any(most > m)) {                   // seldom behind the first tiles
            const float to = lanes_max(most);
            if (m == -INFINITY) sum *= 0.f, a *= 0.f;       // (nothing yet, or a NaN, which stays)
            else {
                const Sums now = moved_to(Sums{m, ones, sum, a}, to);
                sum = now.s, a = now.a;
            }
            ones = 0.f;
            m = to;
        }
        const float from = m == -INFINITY ? 0.f : m;
        if (__any(most == m)) {                  // some term is 1
#pragma unroll
            for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = fmaxf(v[q][e] - from, -3e38f), w = lp_exp(v[q][e] - from);
                    ones += w == 1.f ? 1.f : 0.f;
                    sum += w == 1.f ? 0.f : w;
                    a = fmaf(t, w, a);
                }
        } else {
#pragma unroll
            for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = v[q][e] - from, w = lp_exp(t);
                    sum += w;
                    a = fmaf(fmaxf(t, -3e38f), w, a);      // (minus infinity has no weight; a NaN is in the other sum)
                }
        }
#pragma unroll
        for (int q = 0; q < LP_QUADS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = next[q][e];
    }
    return Sums{m, lanes_sum(ones), lanes_sum(sum), lanes_sum(a)};
}

// A list of candidates that logits join as they come, a lane's each; it keeps the best `top`.
struct Candidates {
    uint64_t* list;                              // LP_LIST + LP_PAD places in LDS
    int top, held = 0;
    float from;                                  // the least logit that joins
    __device__ Candidates(uint64_t* list, int top, float from) : list(list), top(top), from(from) {}
    __device__ void take(float logit, int token, bool there, int lane) {
        bool joins = there && logit >= from;
        uint64_t who = __ballot(joins);
        if (who == 0) return;
        if (held + WAVE > LP_LIST) {             // (then more than `top`)
            put_in_order(list, held, top, lane);
            held = top;
            from = fmaxf(from, logit_of(list[top - 1]));
            joins = there && logit >= from;
            who = __ballot(joins);
        }
        held = append(list, held, who, joins, candidate(logit, token));
    }
    // in order; `last`: what comes from here on has larger numbers, and has to be larger than what is as large as the last place
    __device__ void settle(bool last, int lane) {
        put_in_order(list, held, top, lane);
        held = min(held, top);
        if (last && held == top) from = fmaxf(from, unordered(ordered(logit_of(list[top - 1])) + 1));      // (above infinity: a NaN, which nothing reaches)
    }
};

// The best `top` of a row in order into lists[0], by a block of WAVES waves.  largest: the groups'.  (Every wave calls it; the first one's lanes may read
// the list when it returns.)
template <int WAVES> struct ChosenGroups {
    int chosen[LP_CHOSEN], n, candidates;
    float reached[WAVES];
};
// HOLD: the groups' largest are read once and held (up to LP_GROUPS of them), not read again from LDS.
template <int WAVES, bool HOLD>
__device__ inline void likeliest(const float* largest, int groups, int span, const float* __restrict__ x, int V, int top, uint64_t (*lists)[LP_LIST + LP_PAD],
                                 ChosenGroups<WAVES>& share, int lane, int wave) {
    constexpr int THREADS = WAVES * WAVE, MOST = HOLD ? LP_GROUPS / THREADS : 1;
    const int thread = wave * WAVE + lane;
    float held[MOST], most = -INFINITY;          // the thread's groups: thread, thread + THREADS, ..
    if constexpr (HOLD) {
#pragma unroll
        for (int u = 0; u < MOST; ++u) {
            held[u] = -INFINITY;
            if (u * THREADS < groups) held[u] = largest[min(thread + u * THREADS, groups - 1)];        // (the same in every lane)
        }
#pragma unroll
        for (int u = 0; u < MOST; ++u) {
            if (thread + u * THREADS >= groups) held[u] = -INFINITY;
            most = fmaxf(most, held[u]);
        }
    } else {
        for (int i = thread; i < groups; i += THREADS) most = fmaxf(most, largest[i]);
    }
    if (thread == 0) share.n = share.candidates = 0;
    // what its share of `top` lanes of each wave reach; so the least of that is reached by `top` threads' largest
    const int waves = min(WAVES, (groups + WAVE - 1) / WAVE), of_wave = (top + waves - 1) / waves;
    float reached = INFINITY;
    if (wave < waves) {
        float left = most;
        for (int n = 0; n < of_wave && reached > -INFINITY;) {
            reached = lanes_max(left);
            const bool is = left == reached;
            n += __popcll(__ballot(is));
            left = is ? -INFINITY : left;
        }
    }
    if (lane == 0) share.reached[wave] = reached;
    __syncthreads();
    float from = share.reached[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) from = fminf(from, share.reached[w]);
    if (most >= from) {
        if constexpr (HOLD) {
#pragma unroll
            for (int u = 0; u < MOST; ++u)
                if (held[u] >= from && thread + u * THREADS < groups) {
                    const int at = atomicAdd(&share.n, 1);
                    if (at < LP_CHOSEN) share.chosen[at] = thread + u * THREADS;
                }
        } else {
            for (int i = thread; i < groups; i += THREADS)
                if (largest[i] >= from) {
                    const int at = atomicAdd(&share.n, 1);
                    if (at < LP_CHOSEN) share.chosen[at] = i;
                }
        }
    }
    __syncthreads();
    const int n = share.n, per = span * LP_QUADS * 4;      // groups, and logits of each
    if (n <= LP_CHOSEN) {
        // 16 lanes a group: four groups a wave at once
        auto token_at = [&](int i, int in) {
            const int group = share.chosen[min(i, n - 1)];
            return i < n ? (group / WAVE * span + in / 16) * LP_TILE + in % 16 / 4 * WAVE * 4 + group % WAVE * 4 + in % 4 : V;
        };
        for (int i0 = wave * 4; i0 < n; i0 += WAVES * 4)
            for (int part = 0; part < per; part += 16) {
                const int token = token_at(i0 + lane / 16, part + lane % 16);
                const float logit = x[min(token, V - 1)];
                if (token < V && logit >= from) {
                    const int at = atomicAdd(&share.candidates, 1);
                    if (at < LP_LIST) lists[0][at] = candidate(logit, token);
                }
            }
        __syncthreads();
        if (wave != 0) return;
        if (share.candidates <= LP_LIST) {
            put_in_order(lists[0], share.candidates, top, lane);
            return;
        }
        Candidates all(lists[0], top, from);     // more than the list holds: they join it one after the other
        for (int i0 = 0; i0 < n; i0 += 4)
            for (int part = 0; part < per; part += 16) {
                const int token = token_at(i0 + lane / 16, part + lane % 16);
                all.take(x[min(token, V - 1)], token, token < V, lane);
            }
        all.settle(false, lane);
        return;
    }
    // too many that are equal: the waves go over the row themselves, in order of the numbers
    Candidates mine(lists[wave], top, from);
    const int share_of = (int)(((long long)V + WAVES * WAVE * 4 - 1) / (WAVES * WAVE * 4)) * WAVE * 4;
    const int begin = (int)min((long long)V, (long long)wave * share_of), end = (int)min((long long)V, (long long)begin + share_of);
    for (int at = begin; at < end; at += WAVE * 4) {
        float v[1][4];
        read_tile<1>(x, at, end, lane, v);
        const int held = mine.held;
#pragma unroll
        for (int e = 0; e < 4; ++e) mine.take(v[0][e], at + lane * 4 + e, at + lane * 4 + e < end, lane);
        if (mine.held != held && mine.held >= top) mine.settle(true, lane);
    }
    mine.settle(false, lane);
    __syncthreads();
    if (wave != 0) return;
    int n_list = top;
    for (int w = 1; w < WAVES; ++w) {
        if (n_list + top > LP_LIST) { put_in_order(lists[0], n_list, top, lane); n_list = top; }
        if (lane < top) lists[0][n_list + lane] = lists[w][lane];
        n_list += top;
    }
    put_in_order(lists[0], n_list, top, lane);
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
__global__ __launch_bounds__(LP_ROW_WAVES * WAVE) void logprobs_row_kernel(const float* __restrict__ logits, int V, int span, const int* __restrict__ tokens,
                                                                         int top, float* __restrict__ given, float* __restrict__ entropy, int* __restrict__ ids,
                                                                         float* __restrict__ best) {
    extern __shared__ float largest[];               // the groups'
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? LP_ROW_WAVES : 1][LP_LIST + LP_PAD];
    __shared__ ChosenGroups<TOP ? LP_ROW_WAVES : 1> share;
    __shared__ Sums sums[LP_ROW_WAVES];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), row = blockIdx.x;
    const float* x = logits + (size_t)row * V;
    const Given one(x, tokens, row, V);
    const int border = LP_TILE * span, per = (int)(((long long)V + LP_ROW_WAVES * (long long)border - 1) / (LP_ROW_WAVES * (long long)border)) * border;
    const int begin = (int)min((long long)V, (long long)wave * per), end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = scan<TOP>(x, begin, end, span, largest, lane);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    if constexpr (TOP) likeliest<LP_ROW_WAVES, false>(largest, (V + border - 1) / border * WAVE, span, x, V, top, lists, share, lane, wave);
    if (wave != 0) return;
    const Sums all = of_wave(lane < LP_ROW_WAVES ? sums[lane] : Sums{-INFINITY, 0.f, 0.f, 0.f});
    finish(all, lists[0], one, tokens != nullptr, row, top, given, entropy, ids, best, lane);
}

// Few rows: a wave for each slice of a row, whose sums and groups' largest go to memory, ..
constexpr int LP_SLICE_WAVES = 4;
template <bool TOP>
__global__ __launch_bounds__(LP_SLICE_WAVES * WAVE) void logprobs_slice_kernel(const float* __restrict__ logits, int V, int per, int slices, int span, int groups,
                                                                              Sums* __restrict__ sums, float* __restrict__ largest) {
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int slice = blockIdx.x * LP_SLICE_WAVES + wave, row = blockIdx.y;
    if (slice >= slices) return;
    const int begin = slice * per, end = (int)min((long long)V, (long long)begin + per);
    const Sums mine = scan<TOP>(logits + (size_t)row * V, begin, end, span, largest + (size_t)row * groups, lane);
    if (lane == 0) sums[(size_t)row * slices + slice] = mine;
}
// .. and a block for each row that joins them, LP_EACH slices a lane of its first wave.
constexpr int LP_JOIN_WAVES = 8;
template <bool TOP>
__global__ __launch_bounds__(TOP ? LP_JOIN_WAVES * WAVE : WAVE) void logprobs_join_kernel(const float* __restrict__ logits, int V, int slices, int span,
                                                                                       int groups, const int* __restrict__ tokens, int top,
                                                                                       const Sums* __restrict__ sums, const float* __restrict__ largest,
                                                                                       float* __restrict__ given, float* __restrict__ entropy,
                                                                                       int* __restrict__ ids, float* __restrict__ best) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? LP_JOIN_WAVES : 1][LP_LIST + LP_PAD];
    __shared__ ChosenGroups<TOP ? LP_JOIN_WAVES : 1> share;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), row = blockIdx.x;
    const float* x = logits + (size_t)row * V;
    const Given one(x, tokens, row, V);
    Sums each[LP_EACH];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < LP_EACH; ++k) {
        each[k] = lane + k * WAVE < slices ? sums[(size_t)row * slices + lane + k * WAVE] : Sums{-INFINITY, 0.f, 0.f, 0.f};
        m = fmaxf(m, each[k].m);
    }
    if constexpr (TOP) likeliest<LP_JOIN_WAVES, true>(largest + (size_t)row * groups, groups, span, x, V, top, lists, share, lane, wave);
    if (wave != 0) return;
    Sums all = {m, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < LP_EACH; ++k) {
        const Sums here = moved_to(each[k], m);
        all.ones += here.ones;
        all.s += here.s;
        all.a += here.a;
    }
    finish(of_wave(all), lists[0], one, tokens != nullptr, row, top, given, entropy, ids, best, lane);
}

// Whether each row has a block of its own: short rows, which a block reads as soon as many waves and their joining kernel do, and as many rows as there are
// compute units, nearly.  us in a recorded graph / called one by one, slices and a block a row: 16 rows of 4,000, no alternatives 5.7 / 14.9 and 4.2 / 10.9, five 8.9 / 15.5
// and 6.3 / 11.4; of 16,000, five 10.5 / 15.5 8.6 / 11.5; of 32,000, none 6.1 / 15.0 8.0 / 11.0, five 10.2 / 15.5 11.2 / 11.5; of 50,000, five 10.6 / 15.4 15.5 / 14.8.  100 rows of
// 151,936, none 16.1 / 15.7 25.1 / 24.4, five 21.6 / 21.1 30.1 / 29.6; 250 none 29.9 / 28.3 28.3 / 27.5, five 40.7 / 39.6 33.4 / 32.6.
static bool by_row(int rows, int V, int top) { return V <= 32768 || rows >= (top ? 176 : 240); }
constexpr int LP_WAVES_WANTED = 4096;            // below, slices are as short as it takes for so many waves

static long long tiles_of(int V) { return ((long long)V + LP_TILE - 1) / LP_TILE; }
static int span_of(int V) { return (int)((tiles_of(V) * WAVE + LP_GROUPS - 1) / LP_GROUPS); }          // tiles of a group
static int groups_of(int V) { return (int)((tiles_of(V) + span_of(V) - 1) / span_of(V)) * WAVE; }
// Logits of a slice: whole groups.
static int slice_size(int rows, int V) {
    const long long tiles = tiles_of(V), all = tiles * rows, span = span_of(V);
    const long long least = (tiles + LP_SLICES - 1) / LP_SLICES, wanted = (all + LP_WAVES_WANTED - 1) / LP_WAVES_WANTED;
    return (int)(((least > wanted ? least : wanted) + span - 1) / span * span * LP_TILE);
}
static int slices_of(int rows, int V) { return (int)(((long long)V + slice_size(rows, V) - 1) / slice_size(rows, V)); }

// Bytes of workspace, 0: none is needed.
PALM_API long long palm_token_logprobs_work(int rows, int V, int top) {
    if (rows <= 0 || V <= 0 || by_row(rows, V, top)) return 0;
    return (long long)rows * (slices_of(rows, V) * (long long)sizeof(Sums) + (top ? 4ll * groups_of(V) : 0));
}

// logits [rows, V] float32; tokens [rows] int32 or null; given [rows] (with tokens), entropy [rows], ids and best [rows, top].
PALM_API int palm_token_logprobs(hipStream_t stream, const float* logits, int rows, int V, const int* tokens, int top, void* work, long long work_bytes,
                                 float* given, float* entropy, int* ids, float* best) {
    PALM_CHECK(rows >= 0 && V > 0 && V <= 1 << 30, "token_logprobs: %d rows of %d", rows, V);
    PALM_CHECK(top >= 0 && top <= LP_MOST && top <= V, "token_logprobs: the %d likeliest of %d tokens (%d at most)", top, V, LP_MOST);
    if (rows == 0) return 0;
    PALM_CHECK(work_bytes >= palm_token_logprobs_work(rows, V, top) && (work || work_bytes == 0), "token_logprobs: a workspace of %lld bytes is too small", work_bytes);
    const int span = span_of(V), groups = groups_of(V);
    if (by_row(rows, V, top)) {
        if (top) logprobs_row_kernel<true><<<rows, LP_ROW_WAVES * WAVE, groups * sizeof(float), stream>>>(logits, V, span, tokens, top, given, entropy, ids, best);
        else logprobs_row_kernel<false><<<rows, LP_ROW_WAVES * WAVE, 0, stream>>>(logits, V, span, tokens, top, given, entropy, ids, best);
        PALM_LAUNCHED();
        return 0;
    }
    const int per = slice_size(rows, V), slices = slices_of(rows, V);
    Sums* sums = (Sums*)work;
    float* largest = (float*)(sums + (size_t)rows * slices);
    const dim3 grid((slices + LP_SLICE_WAVES - 1) / LP_SLICE_WAVES, rows);
    if (top) logprobs_slice_kernel<true><<<grid, LP_SLICE_WAVES * WAVE, 0, stream>>>(logits, V, per, slices, span, groups, sums, largest);
    else logprobs_slice_kernel<false><<<grid, LP_SLICE_WAVES * WAVE, 0, stream>>>(logits, V, per, slices, span, groups, sums, largest);
    PALM_LAUNCHED();
    if (top) logprobs_join_kernel<true><<<rows, LP_JOIN_WAVES * WAVE, 0, stream>>>(logits, V, slices, span, groups, tokens, top, sums, largest, given, entropy, ids, best);
    else logprobs_join_kernel<false><<<rows, WAVE, 0, stream>>>(logits, V, slices, span, groups, tokens, top, sums, largest, given, entropy, ids, best);
    PALM_LAUNCHED();
    return 0;
}
