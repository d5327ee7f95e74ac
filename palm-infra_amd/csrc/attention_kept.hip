// Causal grouped-query attention over the paged cache in which a query at position p sees the last `window` positions
// (p - window < j <= p) and its sequence's first `kept` ones (j < kept): all arithmetic in 32-bit, any head size up to 512.  This is the
// float32 mode, and what serves head sizes that the bfloat16 matrix-core kernels do not take.
//
//   s_j = scale q . k_j for the keys seen,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m their maximum
//
// K is [pages, nkv, 64, hd], V is kept transposed, [pages, nkv, hd, 64].  What a run of queries sees is the pages of the first positions
// that lie before the window's first page, then the pages from there on: they are walked as one row.  The pages between are not
// looked at (they may have been given back).
//
// Both products run on the matrix cores in float32 (v_mfma_f32_16x16x4_f32: every product and sum an FMA), transposed as in the
// bfloat16 kernels:  S^T[key, column] = K Q^T,  O^T[d, column] = V^T P^T.  A lane (r, g) holds row r of the first operand and column r of the
// second at the places g of the four summed ones, and rows 4 g .. 4 g + 3 of column r of the result.  So a lane's four scores of a tile of 16 keys are
// of keys 4 g .. 4 g + 3, and the products that follow take them as they are if their first operand is V^T at the same keys: one read of 16 bytes.
// The 16 columns are (position, head): up to 16 heads of the kv head, of as many positions as fit.
//
// A block has four waves that take every fourth page, and a long row is cut into slices of several blocks, joined by a second kernel:
// single tokens and short runs behind a long history have few columns and many pages.
//
// A key that a column does not see has weight zero there, but the products multiply its value all the same, and zero times an infinity or a
// NaN (a page's uncleared end, a token whose activations overflowed and that has left the window) is NaN.  On a page where some column sees
// less than all keys such values are taken as zero, and added again, as they are, to the columns that do see them.
#include "mfma.h"

PALM_DEFINE_LAST_ERROR()

constexpr int KA_WAVES = 4;
constexpr int KA_COLUMNS = 16;
constexpr int KA_MAX_HD = 512;

__device__ inline f32x4 mfma_16x16x4(float a, float b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0); }

// A value the compiler knows nothing of: what is computed from it is computed there, and not kept in registers for the whole kernel.
__device__ inline int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// How a row of a head's elements is read: FULL: hd is all 16 DT of them; FOURS: hd is a multiple of four and rows start on their sizes; ANY.
enum Rows { FULL, FOURS, ANY };

// Four consecutive elements from d on, widened; beyond hd zeros.  Every read is unconditional (an absent one reads what is there and is made zero by a
// select): behind a branch reads would be waited for one by one.
template <Rows ROWS, typename T> __device__ inline f32x4 four_at(const T* row, int d, int hd) {
    f32x4 v;
    if constexpr (ROWS == ANY) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = to_float(row[min(d + e, hd - 1)]);
            v[e] = d + e < hd ? v[e] : 0.f;
        }
        return v;
    } else {
        const T* at = row + (ROWS == FULL ? d : min(d, hd - 4));
        if constexpr (sizeof(T) == 4) {
            const float4 four = *reinterpret_cast<const float4*>(at);
            v = f32x4{four.x, four.y, four.z, four.w};
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(at);
            v = f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
        }
        if constexpr (ROWS != FULL) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = d < hd ? v[e] : 0.f;
        }
        return v;
    }
}

// `places` elements on: the same start in all lanes and an offset of 32 bits, which is how a load takes them without an address of 64 bits
template <typename T> __device__ inline const T* further(const T* start, unsigned places) {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(start) + places * (unsigned)sizeof(T));
}

__device__ inline bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
// e^x for x <= 0 (minus infinity: 0), to 2^-24 |x| and the hardware's 2^x's last place; what is below 2^-126 is zero beside a sum of at least 1
__device__ inline float exp_weight(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// The pages that queries at positions lo .. hi see, as one row of n.
struct SeenRow {
    int n, front, page_lo;       // of the row, the first `front` are the sequence's own first pages, the others the pages from page_lo on
    __device__ SeenRow(int lo, int hi, int window, int kept) {
        page_lo = max(0, lo - window + 1) / PAGE_TOKENS;
        front = min((kept + PAGE_TOKENS - 1) / PAGE_TOKENS, page_lo);
        n = front + hi / PAGE_TOKENS - page_lo + 1;
    }
    __device__ int page(int i) const { return i < front ? i : i - front + page_lo; }
};

// grid (kv heads * groups of heads, tiles of positions, sequences * slices).  A record of the workspace, for each (row, head, slice): maximum, sum, two
// floats unused, then the unnormalised output.
//
// Up to 128 elements a head (AHEAD) a page's keys are asked for together, and its values as the keys' registers come free: a wave has few pages, and
// what it waits for memory is what a short prompt takes.  A page is 256 products of 32 clocks for heads of 128, 3.4 us of a wave.  A prompt of
// 157 tokens, 32 heads of 128 over 8, a window of 64 takes 13.3 us (20.6 with reads behind branches, waited for one by one; 32 with two pages' reads in flight
// and half the waves), 7.7 with heads of 64, 19.5 with heads of 90; 600 tokens with a window of 512: 76 us, 38 TFLOP/s of what is seen.  There the matrix cores
// are at work a quarter of the time (an eighth of it for keys of whole pages that are masked): a SIMD has 1.1 waves in the mean of the two it has places
// for, and a compute unit none for a third of the time, because rows of one to ten pages are dealt to four waves, 1,200 blocks come in 2.3 rounds, and a wave's
// first page is waited for.  Longer heads have no registers for a page ahead and read as they go: heads of 256 take 52 us for the 157 tokens.  One token behind 5,000 in
// a window of 2,048 takes 22 us, 48 of 300 to 9,000 tokens 166.
template <typename T, int DT, Rows ROWS>
__global__ __launch_bounds__(KA_WAVES * WAVE) __attribute__((amdgpu_waves_per_eu(DT <= 8 ? 2 : 1))) void attention_kept_kernel(
    const T* __restrict__ q, const T* __restrict__ k_cache, const T* __restrict__ v_cache, const int* __restrict__ block_table, int max_pages,
    const int* __restrict__ seq_slot, const int* __restrict__ seq_start, const int* __restrict__ seq_new, const int* __restrict__ cu_new, int nh,
    int nkv, int head_size, float scale, int window, int kept, int heads, int slices, float* __restrict__ work, T* __restrict__ out) {
    constexpr bool AHEAD = DT <= 4 || (DT == 8 && ROWS == FULL);       // (more than that is more than the registers hold)
    const int hd = ROWS == FULL ? DT * 16 : head_size;
    __shared__ f32x4 o_lds[KA_WAVES - 1][DT][WAVE];
    __shared__ float m_lds[KA_WAVES - 1][WAVE], l_lds[KA_WAVES - 1][WAVE];
    const int b = blockIdx.z / slices, slice = blockIdx.z % slices;
    const int G = nh / nkv, n_groups = (G + heads - 1) / heads;
    const int kvh = blockIdx.x / n_groups, group = blockIdx.x % n_groups;
    const int here = min(heads, G - group * heads), rows = KA_COLUMNS / heads;      // heads and positions of the tile
    const int n_new = seq_new[b], tile = blockIdx.y * rows;
    if (tile >= n_new) return;
    const int lane = threadIdx.x % WAVE, r = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int start = seq_start[b], last = min(tile + rows, n_new) - 1;
    const int qi = min(tile + r / heads, last);                                     // this lane's column
    const bool valid = r / heads < rows && tile + r / heads <= last && r % heads < here;
    const int head = kvh * G + group * heads + min(r % heads, here - 1);
    const size_t row = (size_t)cu_new[b] + qi;
    const int pos = start + qi, first = max(0, pos - window + 1);
    const SeenRow seen(start + tile, start + last, window, kept);
    const int per = (seen.n + slices - 1) / slices, begin = slice * per, end = min(seen.n, begin + per);
    const int all_first = max(0, start + last - window + 1), all_last = start + tile;   // keys from all_first to all_last: seen by every column
    const int* pages = block_table + (size_t)seq_slot[b] * max_pages;
    auto place = [&](int i) { return ((size_t)__builtin_amdgcn_readfirstlane(pages[seen.page(i)]) * nkv + kvh) * PAGE_TOKENS * hd; };

    f32x4 qv[DT], o[DT], kd[AHEAD ? 4 : 1][DT], vd[AHEAD ? DT : 1][4];
    auto read_key = [&](size_t at, int t, int dt) __attribute__((always_inline)) {
        const T* page = k_cache + at;
        if constexpr (ROWS == FULL) return four_at<FULL>(further(page, ((16 * t + r) * hd + dt * 16 + 4 * g)), 0, hd);
        return four_at<ROWS>(further(page, (16 * t + r) * hd), dt * 16 + 4 * fresh(g), hd);
    };
    auto read_values = [&](size_t at, int dt, f32x4 (&to)[4]) __attribute__((always_inline)) {
        const int d = dt * 16 + (AHEAD ? r : fresh(r));
        const T* page = v_cache + at;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            to[t] = four_at<FULL>(further(page, (ROWS == FULL ? d : min(d, hd - 1)) * PAGE_TOKENS + 16 * t + 4 * g), 0, PAGE_TOKENS);
            if constexpr (ROWS != FULL) {
#pragma unroll
                for (int e = 0; e < 4; ++e) to[t][e] = d < hd ? to[t][e] : 0.f;
            }
        }
    };
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        qv[dt] = four_at<ROWS>(q + (row * nh + head) * hd, dt * 16 + 4 * g, hd);
        o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int i = begin + wave; i < end; i += KA_WAVES) {
        const int key0 = seen.page(i) * PAGE_TOKENS;
        const bool masked = all_last < key0 + PAGE_TOKENS - 1 || (all_first > key0 && kept < key0 + PAGE_TOKENS);   // the same in every lane
        const size_t at = place(i);
        if constexpr (AHEAD) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) kd[t][dt] = read_key(at, t, dt);
            __builtin_amdgcn_sched_barrier(0);
        }
        // (no && or ||: a select, not a branch for every key)
        auto sees = [&](int in_page) { const int key = key0 + in_page; return (key <= pos) & ((key >= first) | (key < kept)); };
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if constexpr (!AHEAD)
                    if (dt % 8 == 0) {
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int x = dt; x < dt + 8 && x < DT; ++x) kd[0][x] = read_key(at, t, x);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = mfma_16x16x4(kd[AHEAD ? t : 0][dt][e], qv[dt][e], acc);
            }
            s[t] = acc * scale;
            if constexpr (AHEAD) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    if (dt * 4 / DT == t - 1 || (t == 3 && dt * 4 / DT == 3)) read_values(at, dt, vd[dt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = sees(16 * t + 4 * g + e) ? s[t][e] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[t][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        const float m_new = fmaxf(m, mx), from = m_new == -INFINITY ? 0.f : m_new;      // (a column may see no key of its tile's first pages)
        const float alpha = exp_weight(m - from);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] = exp_weight(s[t][e] - from);
                l += s[t][e];
            }
        float wild = 0.f;                                       // a NaN: the page has values that are none
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f32x4 acc = o[dt] * alpha;
            f32x4 (&v_of)[4] = vd[AHEAD ? dt : 0];
            if constexpr (!AHEAD) {
                if (dt % 2 == 0) __builtin_amdgcn_sched_barrier(0);     // (two tiles' values at a time: the outputs need the registers)
                read_values(at, dt, v_of);
            }
            if (masked) {
                float odd = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd = fmaf(v_of[t][e], 0.f, odd);
                if (__any(odd != 0.f)) {
                    wild = NAN;
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v_of[t][e] = finite(v_of[t][e]) ? v_of[t][e] : 0.f;
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = mfma_16x16x4(v_of[t][e], s[t][e], acc);
            o[dt] = acc;
        }
        if (wild != 0.f) {                                      // (the same in every lane)
            for (int j = 0; j < PAGE_TOKENS; ++j) {
                const bool seen_here = sees(j);
                const int d0 = AHEAD ? 4 * g : fresh(4 * g);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = dt * 16 + d0 + e;
                        const float v = to_float(v_cache[at + (size_t)min(d, hd - 1) * PAGE_TOKENS + j]);
                        o[dt][e] += seen_here & !finite(v) & (d < hd) ? v : 0.f;
                    }
            }
        }
    }
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (wave > 0) {
        m_lds[wave - 1][lane] = m;
        l_lds[wave - 1][lane] = l;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o_lds[wave - 1][dt][lane] = o[dt];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < KA_WAVES - 1; ++w) {
        const float mw = m_lds[w][lane], lw = l_lds[w][lane], top = fmaxf(m, mw);
        if (mw == -INFINITY && lw == 0.f) continue;             // it saw none of the column's keys (with scores that are all NaN its sum is one, and shows)
        const float mine = exp_weight(m - top), its = exp_weight(mw - top);
        l = l * mine + lw * its;
        m = top;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = o[dt] * mine + o_lds[w][dt][lane] * its;
    }
    if (!valid) return;
    if (slices > 1) {
        float* record = work + ((row * nh + head) * slices + slice) * (hd + 4);
        if (g == 0) { record[0] = m; record[1] = l; }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (dt * 16 + 4 * g + e < hd) record[4 + dt * 16 + 4 * g + e] = o[dt][e];
        return;
    }
    T* to = out + (row * nh + head) * hd;
    const float inv = 1.0f / l;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int d = dt * 16 + 4 * g;
        if constexpr (ROWS == FULL && sizeof(T) == 4) {
            *reinterpret_cast<float4*>(to + d) = make_float4(o[dt][0] * inv, o[dt][1] * inv, o[dt][2] * inv, o[dt][3] * inv);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < hd) to[d + e] = from_float<T>(o[dt][e] * inv);
        }
    }
}

// A wave for each (row, head): the slices' records in their order.
template <typename T>
__global__ __launch_bounds__(WAVE) void attention_kept_join_kernel(const float* __restrict__ work, int slices, int hd, T* __restrict__ out) {
    const float* w = work + (size_t)blockIdx.x * slices * (hd + 4);
    const int lane = threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (int s = lane; s < slices; s += WAVE) m = fmaxf(m, w[(size_t)s * (hd + 4)]);
    m = wave_max(m);
    for (int s = lane; s < slices; s += WAVE) l += w[(size_t)s * (hd + 4) + 1] * exp_weight(w[(size_t)s * (hd + 4)] - m);
    l = wave_sum(l);
    for (int d = lane; d < hd; d += WAVE) {
        float o = 0.f;
#pragma unroll 8
        for (int s = 0; s < slices; ++s) {
            const float ms = w[(size_t)s * (hd + 4)], v = w[(size_t)s * (hd + 4) + 4 + d];
            o += ms == -INFINITY ? 0.f : v * exp_weight(ms - m);       // (an empty slice has no output)
        }
        out[(size_t)blockIdx.x * hd + d] = from_float<T>(o / l);
    }
}

// heads of a kv head that a tile's columns are
static int heads_of_tile(int nh, int nkv) { return nh / nkv < KA_COLUMNS ? nh / nkv : KA_COLUMNS; }

// Into how many slices a row of pages is cut: until the launch has two blocks a compute unit, and not into less than a page for each wave.
PALM_API int palm_attention_kept_slices(int n_seqs, int max_new, int max_total, int nh, int nkv, int window, int kept) {
    PALM_CHECK(n_seqs > 0 && max_new > 0 && max_total >= max_new && nh > 0 && nkv > 0 && nh % nkv == 0 && window > 0 && kept >= 0,
               "attention_kept: seqs=%d max_new=%d max_total=%d heads=%d kv=%d window=%d kept=%d", n_seqs, max_new, max_total, nh, nkv, window, kept);
    const int heads = heads_of_tile(nh, nkv), rows = KA_COLUMNS / heads;
    const long long blocks = (long long)nkv * ((nh / nkv + heads - 1) / heads) * ((max_new + rows - 1) / rows) * n_seqs;
    const long long keys = (long long)window + rows + kept < max_total ? (long long)window + rows + kept : max_total;
    const long long most = ((keys + PAGE_TOKENS - 1) / PAGE_TOKENS + KA_WAVES - 1) / KA_WAVES, wanted = (512 + blocks - 1) / blocks;
    return (int)(wanted < most ? wanted : most);
}

// dtype of q, the cache and out: 0 float32, 1 bfloat16.  work: rows * nh * slices * (hd + 4) floats where there is more than one slice.
PALM_API int palm_attention_kept(hipStream_t stream, const void* q, int dtype, const void* k_cache, const void* v_cache, const int* block_table,
                                 int max_pages, const int* seq_slot, const int* seq_start, const int* seq_new, const int* cu_new, int n_seqs, int rows,
                                 int max_new, int nh, int nkv, int hd, float scale, int window, int kept, int slices, float* work, void* out) {
    PALM_CHECK(n_seqs >= 0 && max_new >= 0 && rows >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0, "attention_kept: seqs=%d max_new=%d heads=%d kv=%d", n_seqs,
               max_new, nh, nkv);
    PALM_CHECK(hd > 0 && hd <= KA_MAX_HD, "attention_kept: head size %d is not within 1 to %d", hd, KA_MAX_HD);
    PALM_CHECK(window > 0 && kept >= 0 && max_pages > 0, "attention_kept: window=%d kept=%d max_pages=%d", window, kept, max_pages);
    PALM_CHECK(slices >= 1 && (slices == 1 || work), "attention_kept: %d slices need a workspace", slices);
    if (n_seqs == 0 || max_new == 0 || rows == 0) return 0;
    const int heads = heads_of_tile(nh, nkv), per = KA_COLUMNS / heads;
    const long long x = (long long)nkv * ((nh / nkv + heads - 1) / heads), y = (max_new + per - 1) / per, z = (long long)n_seqs * slices;
    PALM_CHECK(y <= 65535 && z <= 65535, "attention_kept: %d new tokens of %d sequences in %d slices are more than one launch takes", max_new, n_seqs, slices);
    const dim3 grid((unsigned)x, (unsigned)y, (unsigned)z);
    const bool fours = hd % 4 == 0 && ((uintptr_t)q | (uintptr_t)k_cache) % 16 == 0;
    PALM_CHECK((uintptr_t)v_cache % 16 == 0 && (uintptr_t)out % 16 == 0, "attention_kept: values or results do not start on 16 bytes");
#define PALM_KEPT(DT, ROWS) attention_kept_kernel<T, DT, ROWS><<<grid, KA_WAVES * WAVE, 0, stream>>>((const T*)q, (const T*)k_cache, (const T*)v_cache, \
        block_table, max_pages, seq_slot, seq_start, seq_new, cu_new, nh, nkv, hd, scale, window, kept, heads, slices, work, (T*)out)
    PALM_DTYPE_SWITCH(dtype, T,
        if (!fours) { if (hd <= 128) PALM_KEPT(8, ANY); else PALM_KEPT(32, ANY); }
        else if (hd == 64) PALM_KEPT(4, FULL);
        else if (hd == 128) PALM_KEPT(8, FULL);
        else if (hd <= 32) PALM_KEPT(2, FOURS);
        else if (hd <= 64) PALM_KEPT(4, FOURS);
        else if (hd <= 128) PALM_KEPT(8, FOURS);
        else if (hd <= 256) PALM_KEPT(16, FOURS);
        else PALM_KEPT(32, FOURS);
        PALM_LAUNCHED();
        if (slices > 1) { attention_kept_join_kernel<T><<<rows * nh, WAVE, 0, stream>>>(work, slices, hd, (T*)out); PALM_LAUNCHED(); });
#undef PALM_KEPT
    return 0;
}
