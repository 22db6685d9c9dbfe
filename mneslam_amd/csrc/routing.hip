// routing.hip -- tokens (points, samples) sorted by expert, dealt to the experts' rows, and blended back with weights.
//
//   slot n k_max + k holds the expert ids[n][k] of token n; ids outside 0 .. experts - 1 name no expert
//   sort      a stable counting sort of the slots by expert: order[row] = slot, position[slot] = row, offsets[e] = first row of expert e
//   dispatch  out[position[n][k]] = x[n]                                  dx[n] = sum_k dout[position[n][k]]      (combine, no weights)
//   combine   out[n] = sum_k w[n][k] y[position[n][k]]                    dy[position[n][k]] = w[n][k] dout[n],  dw[n][k] = <dout[n], y[position[n][k]]>
//
// The row movements are bound by memory: 131071 tokens x 4 rows of 2048 bf16 are dealt out in 500 us (2.7 GB, 5.4 TB/s) and combined in 435
// (6.1 TB/s), 16384 x 2 rows of 1024 bf16 in 17 and 16 us, their gradients in 16 and 28 us (166 MB, 5.9 TB/s); rows whose length is no
// multiple of a line at 4 to 5 TB/s (275200 rows of 65 fp32: 37, 36, 36 and 48 us).
//
// A row of the sorted side belongs to one slot, so nothing is added up across workgroups: no atomics on results, and the same bits
// every time.  Sums are fp32 over k = 0, 1, ... (and over a row in a fixed order); a 16-bit result is rounded to nearest even once.
#include "mne_device.h"
#include "mne_elem.h"
#include "mne_launch.h"

#define EX_THREADS 256
#define EX_WAVES (EX_THREADS / 64)
#define EX_CHUNKS 512                               // workgroups of the long form at most
#define EX_SHORT 4096                               // slots up to which one workgroup of 1024 does it all
#define EX_SHORT_EXPERTS 2000                       // its counters of 16 waves fit the LDS
#define EX_SUMS_MOST 16384                          // counters that every workgroup may add up itself
#define EX_AHEAD 8                                  // ids that a lane loads before it looks at the first

// ---- sort ------------------------------------------------------------------------------------------------------------
// Bound by launches and round trips to memory, not by bytes.  Three forms (us, 8 / 129 / 1000 experts, one choice each):
//   slots                                     512                4096               32768              524288
//   one workgroup                             3.6 / 4.0 / 5.2    6.1 / 7.0 / 8.6    (16384: 16 / 20 / 23)
//   count, place with the sums in it          6.4 / 6.8 / -      6.5 / 7.7 / -      6.9 / 15.2* / -    11.7 / - / -
//   count, scan, place                        10.2 / 10.7 / 13.1 10.4 / 11.1 / 13.8 10.7 / 11.7 / 13.9 14.5 / 16.4 / 21.5
// so: one workgroup up to 4096 slots, else sums in place up to 16384 counters (* : beyond them), else a scan of its own.
__device__ __forceinline__ int ex_id(const ExpertSortArgs& a, int slot) {        // what names no expert sorts behind all of them
    const long long e = a.wide ? ((const long long*)a.ids)[slot] : ((const int*)a.ids)[slot];
    return e >= 0 && e < a.experts ? (int)e : a.experts;
}

// the slots first + 64 j + lane of a wave, j = 0 .. EX_AHEAD - 1, at most `last`: loaded together, looked at one after the other
__device__ __forceinline__ void ex_ids(const ExpertSortArgs& a, long long first, long long last, int* e) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < EX_AHEAD; ++j) {
        const long long slot = first + 64 * j + lane;
        e[j] = slot < last ? ex_id(a, (int)slot) : -1;
    }
}

// e: the ids of the first EX_AHEAD x 64 slots, loaded before
__device__ __forceinline__ void ex_count(const ExpertSortArgs& a, long long first, long long last, const int* e, int* cnt) {
#pragma unroll
    for (int j = 0; j < EX_AHEAD; ++j)
        if (e[j] >= 0) atomicAdd(&cnt[e[j]], 1);
    for (long long j0 = first + 64 * EX_AHEAD; j0 < last; j0 += 64 * EX_AHEAD) {
        int more[EX_AHEAD];
        ex_ids(a, j0, last, more);
#pragma unroll
        for (int j = 0; j < EX_AHEAD; ++j)
            if (more[j] >= 0) atomicAdd(&cnt[more[j]], 1);
    }
}

__global__ __launch_bounds__(EX_THREADS) void expert_count_kernel(ExpertSortArgs a) {
    MNE_DYN_LDS(lds);
    int* cnt = (int*)lds;
    const long long first = ((long long)blockIdx.x * EX_WAVES + (threadIdx.x >> 6)) * a.per_wave;
    const long long last = first + a.per_wave < a.m ? first + a.per_wave : a.m;
    int ids[EX_AHEAD];
    ex_ids(a, first, last, ids);
    for (int e = threadIdx.x; e <= a.experts; e += EX_THREADS) cnt[e] = 0;
    __syncthreads();
    ex_count(a, first, last, ids, cnt);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += EX_THREADS) a.count[(long long)blockIdx.x * (a.experts + 1) + e] = cnt[e];
}

// count[chunk][e] becomes the number of e's slots in the chunks before, total[e] the number in all: 64 experts a workgroup, a
// sixteenth of the chunks (32 at most) a wave, in registers between the two passes
__global__ __launch_bounds__(1024) void expert_scan_kernel(ExpertSortArgs a) {
    __shared__ int part[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = (int)blockIdx.x * 64 + lane, stride = a.experts + 1;
    const int each = (a.chunks + 15) / 16, lo = w * each, hi = lo + each < a.chunks ? lo + each : a.chunks;
    int c[EX_CHUNKS / 16], sum = 0;
#pragma unroll
    for (int i = 0; i < EX_CHUNKS / 16; ++i) c[i] = e <= a.experts && lo + i < hi ? a.count[(long long)(lo + i) * stride + e] : 0;
#pragma unroll
    for (int i = 0; i < EX_CHUNKS / 16; ++i) sum += c[i];
    part[w][lane] = sum;
    __syncthreads();
    int run = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i < w) run += part[i][lane];
        all += part[i][lane];
    }
#pragma unroll
    for (int i = 0; i < EX_CHUNKS / 16; ++i) {
        if (e <= a.experts && lo + i < hi) a.count[(long long)(lo + i) * stride + e] = run;
        run += c[i];
    }
    if (e <= a.experts && w == 0) a.total[e] = all;
}

// Rows of a workgroup's slots: WAVES waves of a.per_wave consecutive slots.  How many slots of an expert there are in all, and in the
// workgroups before: EX_ALONE, there is one workgroup; EX_SCANNED, expert_scan_kernel has added them up; EX_SUMS, every workgroup adds
// all counters up itself, which is less than another launch as long as they are few.
enum { EX_ALONE, EX_SCANNED, EX_SUMS };
template <int WAVES, int HOW>
__global__ __launch_bounds__(WAVES * 64) void expert_place_kernel(ExpertSortArgs a) {
    constexpr bool ALONE = HOW == EX_ALONE;
    MNE_DYN_LDS(lds);
    int* cnt = (int*)lds;                           // [WAVES][experts + 1]: counters, then next rows
    __shared__ int part[WAVES], sums[HOW == EX_SUMS ? 2 * EX_THREADS : 1];
    const int bins = a.experts + 1, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int* mine = cnt + w * bins;
    const long long first = ((long long)blockIdx.x * WAVES + w) * a.per_wave;
    const long long last = first + a.per_wave < a.m ? first + a.per_wave : a.m;
    int ids[EX_AHEAD];                              // on their way while the counters are cleared and added up
    ex_ids(a, first, last, ids);
    for (int e = threadIdx.x; e < WAVES * bins; e += WAVES * 64) cnt[e] = 0;
    if (HOW == EX_SUMS) {                           // lane e of every `span` has expert e, the spans share the chunks
        int span = 1;
        while (span < bins) span <<= 1;
        const int e = threadIdx.x & (span - 1), at = threadIdx.x / span, step = EX_THREADS / span;
        int before = 0, all = 0;
        if (e < bins)
            for (int c0 = at; c0 < a.chunks; c0 += 8 * step) {
                int x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = c0 + i * step < a.chunks ? a.count[(long long)(c0 + i * step) * bins + e] : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    all += x[i];
                    before += c0 + i * step < (int)blockIdx.x ? x[i] : 0;
                }
            }
        sums[2 * threadIdx.x] = before;
        sums[2 * threadIdx.x + 1] = all;
        __syncthreads();
        before = all = 0;
        if ((int)threadIdx.x < bins)
            for (int i = 0; i < step; ++i) {
                before += sums[2 * (i * span + threadIdx.x)];
                all += sums[2 * (i * span + threadIdx.x) + 1];
            }
        __syncthreads();
        if ((int)threadIdx.x < bins) { sums[2 * threadIdx.x] = before; sums[2 * threadIdx.x + 1] = all; }
    }
    __syncthreads();
    ex_count(a, first, last, ids, mine);
    __syncthreads();
    // first row of every expert: a thread has a run of them, the threads' sums are scanned
    const int each = (bins + WAVES * 64 - 1) / (WAVES * 64), lo = threadIdx.x * each, hi = lo + each < bins ? lo + each : bins;
    int sum = 0;
    for (int e = lo; e < hi; ++e) {
        int t = 0;
        if (ALONE) for (int i = 0; i < WAVES; ++i) t += cnt[i * bins + e];
        else t = HOW == EX_SUMS ? sums[2 * e + 1] : a.total[e];
        sum += t;
    }
    int scan = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 63) part[w] = scan;
    __syncthreads();
    int row = scan - sum;
    for (int i = 0; i < w; ++i) row += part[i];
    for (int e = lo; e < hi; ++e) {
        if (blockIdx.x == 0) a.offsets[e] = row;    // (the entry behind the last expert: the number of live rows)
        int t = 0, next = ALONE ? row : row + (HOW == EX_SUMS ? sums[2 * e] : a.count[(long long)blockIdx.x * bins + e]);
        for (int i = 0; i < WAVES; ++i) {
            const int c = cnt[i * bins + e];
            cnt[i * bins + e] = next;
            next += c;
            t += c;
        }
        row += ALONE ? t : HOW == EX_SUMS ? sums[2 * e + 1] : a.total[e];
    }
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < bins) ++bits;
    for (long long j0 = first; j0 < last; j0 += 64 * EX_AHEAD) {
        if (j0 > first || last - first > 64 * EX_AHEAD) ex_ids(a, j0, last, ids);
        for (int j = 0; j < EX_AHEAD && j0 + 64 * j < last; ++j) {        // 64 slots at a time, in order
            int e = -1;
#pragma unroll
            for (int i = 0; i < EX_AHEAD; ++i) e = i == j ? ids[i] : e;
            const bool live = e >= 0;
            const int key = live ? e : a.experts;
            unsigned long long peers = __ballot(live);                    // the lanes with the same expert
            for (int b = 0; b < bits; ++b) {
                const unsigned long long set = __ballot((key >> b) & 1);
                peers &= (key >> b) & 1 ? set : ~set;
            }
            const int before = __popcll(peers & ((1ull << lane) - 1ull)), all = __popcll(peers);
            const int start = mine[key];
            MNE_WAVE_SYNC();
            if (live) {
                const int slot = (int)(j0 + 64 * j) + lane, r = start + before;
                const bool named = e < a.experts;
                if (before == all - 1) mine[e] = r + 1;
                a.position[slot] = named ? r : -1;
                a.order[r] = named ? slot : -1;
            }
            MNE_WAVE_SYNC();
        }
    }
}

// Slots of a wave of the long form, in 64s: as few as make 512 workgroups, and so many that a workgroup's counters are not more than
// twice its slots.
static int ex_per_wave(long long m, int experts) {
    const long long by_size = (m + EX_CHUNKS * EX_THREADS - 1) / (EX_CHUNKS * EX_THREADS), by_experts = (experts + 2 * EX_THREADS) / (2 * EX_THREADS);
    return (int)(64 * (by_size > by_experts ? by_size : by_experts));
}
static int ex_chunks(long long m, int experts) {
    const long long chunk = (long long)EX_WAVES * ex_per_wave(m, experts);
    return m ? (int)((m + chunk - 1) / chunk) : 1;          // (one without slots writes the offsets)
}
static bool ex_sums(long long m, int experts) {
    int span = 1;
    while (span < experts + 1) span <<= 1;
    return span <= EX_THREADS && (long long)ex_chunks(m, experts) * span <= EX_SUMS_MOST;
}
static bool ex_short(long long m, int experts) { return m <= EX_SHORT && experts <= EX_SHORT_EXPERTS; }

long long mne_expert_workspace_ints(long long m, int experts) {
    return ex_short(m, experts) ? 0 : ((long long)ex_chunks(m, experts) + 1) * (experts + 1);
}

int mne_launch_expert_sort(ExpertSortArgs a, void* workspace, hipStream_t st) {
    const int bins = a.experts + 1;
    if (ex_short(a.m, a.experts)) {
        a.per_wave = (int)(((a.m + 15) / 16 + 63) / 64 * 64);
        const size_t lds = (size_t)16 * bins * sizeof(int);
        MNE_SET_MAX_LDS((expert_place_kernel<16, EX_ALONE>), lds);
        MNE_LAUNCH((expert_place_kernel<16, EX_ALONE>), 1, 1024, lds, st, a);
        return 0;
    }
    a.chunks = ex_chunks(a.m, a.experts);
    a.per_wave = ex_per_wave(a.m, a.experts);
    a.count = (int*)workspace;
    a.total = a.count + (long long)a.chunks * bins;
    MNE_LAUNCH(expert_count_kernel, a.chunks, EX_THREADS, bins * sizeof(int), st, a);
    const size_t lds = (size_t)EX_WAVES * bins * sizeof(int);
    if (ex_sums(a.m, a.experts)) {
        MNE_LAUNCH((expert_place_kernel<EX_WAVES, EX_SUMS>), a.chunks, EX_THREADS, lds, st, a);
        return 0;
    }
    MNE_LAUNCH(expert_scan_kernel, (bins + 63) / 64, 1024, 0, st, a);
    MNE_SET_MAX_LDS((expert_place_kernel<EX_WAVES, EX_SCANNED>), lds);
    MNE_LAUNCH((expert_place_kernel<EX_WAVES, EX_SCANNED>), a.chunks, EX_THREADS, lds, st, a);
    return 0;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// A row is cut into columns of P bytes: 16, or where it has fewer the largest power of two it has.  The last column ends where the row
// ends, over a part of the one before it if it must: what two lanes read and write there is the same.  Columns are loaded and stored
// whole whatever their alignment (global memory takes them in one piece; element by element, odd widths would take eight times the
// instructions).  PAST: see ex_past.
typedef unsigned ex_words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned ex_words2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned ex_words1 __attribute__((aligned(2)));
template <int P> struct ExWords;
template <> struct ExWords<16> { typedef ex_words4 mem; typedef unsigned reg __attribute__((ext_vector_type(4))); };
template <> struct ExWords<8> { typedef ex_words2 mem; typedef unsigned reg __attribute__((ext_vector_type(2))); };
template <> struct ExWords<4> { typedef ex_words1 mem; typedef unsigned reg; };
template <> struct ExWords<2> { typedef unsigned short mem; typedef unsigned short reg; };

template <int T, int P, int PAST> struct ExCol {
    typedef typename MneElem<T>::mem elem;
    typedef typename MneWord<sizeof(elem)>::type word;
    typedef typename ExWords<P>::mem mem;
    static constexpr int N = P / (int)sizeof(elem);
    typename ExWords<P>::reg v;
    static __device__ __forceinline__ int start(int c, int width) { return c * N < width - N ? c * N : width - N; }
    __device__ __forceinline__ void clear() { v = (typename ExWords<P>::reg)(0u); }
    __device__ __forceinline__ void load(const char* row, int c, int width) {
        const mem* p = (const mem*)((const elem*)row + start(c, width));
        if (PAST == 2) v = __builtin_nontemporal_load(p);
        else v = *p;
    }
    __device__ __forceinline__ void store(char* row, int c, int width) const {
        mem* p = (mem*)((elem*)row + start(c, width));
        if (PAST) __builtin_nontemporal_store(v, p);
        else *p = v;
    }
    __device__ __forceinline__ unsigned at(int i) const {            // 32 bits of it
        if constexpr (P >= 8) return v[i];
        else return v;
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(elem) == 4) return __uint_as_float(at(j));
        else return MneElem<T>::get(__builtin_bit_cast(elem, (word)(at(j >> 1) >> (j & 1 ? 16 : 0))));
    }
    __device__ __forceinline__ void put(const float* x) {
        if constexpr (P == 2) v = __builtin_bit_cast(word, MneElem<T>::put(x[0]));
        else {
#pragma unroll
            for (int i = 0; i < P / 4; ++i) {
                unsigned u;
                if constexpr (sizeof(elem) == 4) u = __float_as_uint(x[i]);
                else u = (unsigned)__builtin_bit_cast(word, MneElem<T>::put(x[2 * i])) | (unsigned)__builtin_bit_cast(word, MneElem<T>::put(x[2 * i + 1])) << 16;
                if constexpr (P >= 8) v[i] = u;
                else v = u;
            }
        }
    }
};

// a slot's row, -1 where it has none (or the plan's entry is none of a plan's)
__device__ __forceinline__ int ex_row(const ExpertRowArgs& a, long long slot) {
    const int row = a.position[slot];
    return (long long)row < (long long)a.n * a.k ? row : -1;
}

// GROUP lanes have a token and a tile of GROUP * U columns.
template <int T, int P, int U, int PAST>
__global__ __launch_bounds__(EX_THREADS) void expert_dispatch_kernel(ExpertRowArgs a, int group) {
    typedef ExCol<T, P, PAST> Col;
    const long long unit = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    if (unit >= (long long)a.n * a.tiles) return;
    const int n = (int)(unit / a.tiles), c0 = (int)(unit % a.tiles) * group * U + l;
    const long long size = (long long)a.width * sizeof(typename Col::elem), slot = (long long)n * a.k;
    const int total = *a.total;
    Col x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (c0 + u * group < a.cols) x[u].load((const char*)a.a + n * a.a_stride, c0 + u * group, a.width);
    for (int k = 0; k < a.k; ++k) {
        const int row = ex_row(a, slot + k);
        if (row >= 0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * group < a.cols) x[u].store((char*)a.out + row * size, c0 + u * group, a.width);
        }
        if (slot + k >= total) {                    // a row behind the live ones: zero
            Col zero;
            zero.clear();
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * group < a.cols) zero.store((char*)a.out + (slot + k) * size, c0 + u * group, a.width);
        }
    }
}

template <int T, int P, int U, int PAST>
__global__ __launch_bounds__(EX_THREADS) void expert_combine_kernel(ExpertRowArgs a, int group) {
    typedef ExCol<T, P, PAST> Col;
    const long long unit = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    if (unit >= (long long)a.n * a.tiles) return;
    const int n = (int)(unit / a.tiles), c0 = (int)(unit % a.tiles) * group * U + l;
    const long long size = (long long)a.width * sizeof(typename Col::elem), slot = (long long)n * a.k;
    float acc[U][Col::N] = {};
    for (int k = 0; k < a.k; k += 2) {              // two rows in flight
        int row[2];
        float w[2];
        Col y[2][U];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool on = k + i < a.k;
            row[i] = on ? ex_row(a, slot + k + i) : -1;
            w[i] = on && a.weights ? a.weights[slot + k + i] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                y[i][u].clear();
                if (row[i] >= 0 && c0 + u * group < a.cols) y[i][u].load((const char*)a.a + row[i] * a.a_stride, c0 + u * group, a.width);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (row[i] < 0) continue;               // (its weight may be anything)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < Col::N; ++j) acc[u][j] = fmaf(w[i], y[i][u].get(j), acc[u][j]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (c0 + u * group < a.cols) {
            Col o;
            o.put(acc[u]);
            o.store((char*)a.out + n * size, c0 + u * group, a.width);
        }
}

// GROUP lanes have a token: its row of dout against its rows of y, K slots and U columns of a lane at a time.
template <int T, int P, int K, int U, int PAST>
__global__ __launch_bounds__(EX_THREADS) void expert_combine_backward_kernel(ExpertRowArgs a, int group) {
    typedef ExCol<T, P, PAST> Col;
    const long long n = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    const bool there = n < a.n;                     // (all lanes stay: they add up the dot products together)
    const long long size = (long long)a.width * sizeof(typename Col::elem), slot = n * a.k;
    const int total = *a.total;
    for (int k0 = 0; k0 < a.k; k0 += K) {
        int row[K];
        float w[K], dot[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool on = there && k0 + i < a.k;
            row[i] = on ? ex_row(a, slot + k0 + i) : -1;
            w[i] = on && a.weights ? a.weights[slot + k0 + i] : 1.0f;
            dot[i] = 0.0f;
        }
        if (there)
            for (int c0 = l; c0 < a.cols; c0 += group * U) {
                Col d[U], y[K][U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    d[u].clear();
                    if (c0 + u * group < a.cols) d[u].load((const char*)a.a + n * a.a_stride, c0 + u * group, a.width);
                }
                if (a.dw) {
#pragma unroll
                    for (int i = 0; i < K; ++i)
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            y[i][u].clear();
                            if (row[i] >= 0 && c0 + u * group < a.cols) y[i][u].load((const char*)a.b + row[i] * a.b_stride, c0 + u * group, a.width);
                        }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int c = c0 + u * group, twice = c * Col::N - Col::start(c, a.width);     // elements that the column before has
#pragma unroll
                        for (int j = 0; j < Col::N; ++j) {
                            const float x = d[u].get(j);
#pragma unroll
                            for (int i = 0; i < K; ++i) {           // (left out, not multiplied by zero: y may be infinite there)
                                const float more = fmaf(x, y[i][u].get(j), dot[i]);
                                dot[i] = j >= twice ? more : dot[i];
                            }
                        }
                    }
                }
                if (a.out) {
#pragma unroll
                    for (int i = 0; i < K; ++i)
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            if (c0 + u * group >= a.cols) continue;
                            if (row[i] >= 0) {
                                Col o;
                                float x[Col::N];
#pragma unroll
                                for (int j = 0; j < Col::N; ++j) x[j] = w[i] * d[u].get(j);
                                o.put(x);
                                o.store((char*)a.out + row[i] * size, c0 + u * group, a.width);
                            }
                            if (k0 + i < a.k && slot + k0 + i >= total) {
                                Col zero;
                                zero.clear();
                                zero.store((char*)a.out + (slot + k0 + i) * size, c0 + u * group, a.width);
                            }
                        }
                }
            }
        if (a.dw) {
#pragma unroll
            for (int i = 0; i < K; ++i) {
                for (int s = group >> 1; s; s >>= 1) dot[i] += __shfl_xor(dot[i], s);
                if (there && l == 0 && k0 + i < a.k) a.dw[slot + k0 + i] = row[i] >= 0 ? dot[i] : 0.0f;
            }
        }
    }
}

static long long ex_row_bytes(const ExpertRowArgs& a, int type) { return (long long)a.width * (type == MNE_T_F32 ? 4 : 2); }
static int ex_piece(const ExpertRowArgs& a, int type) {
    const long long size = ex_row_bytes(a, type);
    return size >= 16 ? 16 : size >= 8 ? 8 : size >= 4 ? 4 : 2;
}

// Lanes of a token (a power of two, at most a wave, no fewer than make a 128-byte line where there are as many columns) and columns of
// a lane (1 to `most`): of the forms that leave the fewest lanes without a column the one with most columns a lane, whose loads are in
// flight together.  Where that leaves the machine without waves, one column a lane.
struct ExForm { int group, u; };
static ExForm ex_form(ExpertRowArgs& a, int type, int most) {
    const int piece = ex_piece(a, type);
    a.cols = (int)((ex_row_bytes(a, type) + piece - 1) / piece);
    if ((long long)a.n * a.cols < 1 << 17 || piece < 16) most = 1;
    ExForm best = {64, most};
    long long least = 1ll << 62;
    for (int u = 1; u <= most; ++u) {
        int group = 1;
        while (group < 64 && group * u < a.cols) group <<= 1;
        if (group < 8 && u > 1) continue;
        const long long used = ((long long)a.cols + group * u - 1) / (group * u) * (group * u);
        if (used <= least) { least = used; best = {group, u}; }
    }
    a.tiles = (a.cols + best.group * best.u - 1) / (best.group * best.u);
    return best;
}
// workgroups, 0 if there are too many (the threads of a launch are counted in 32 bits)
static unsigned ex_grid(long long units, int group) {
    const long long blocks = (units * group + EX_THREADS - 1) / EX_THREADS;
    return blocks * EX_THREADS <= 0xFFFFFFFFll ? (unsigned)blocks : 0u;
}

// What goes past the caches (PAST): 0 nothing, 1 what is written, 2 what is read as well.
// Written: rows of whole 128-byte lines only -- 32768 rows of 2 KB combined 16 us instead of 30, dealt out 17 instead of 22; with rows of
// 260 bytes, whose lines are written by two, 61 us instead of 36.
// (Combined rows lie one after the other, and still: rows of 64 bytes 69 us and 67 without, of 32 bytes 98 and 78.)
// Dealt-out rows only below 1 GB in all: rows of 4 KB, four to a token, 0.5 GB 108 us instead of 121, but 1 GB 254 instead of 249, 2.1 GB
// 510 instead of 502, 4.3 GB 1025 instead of 1016 (one or two to a token: within 1 % from 0.5 GB on).
// Read: combined rows of 128 MB and more in all, half of what the last cache holds: 128 MB 31 us instead of 33, 2.1 GB 429 instead of 464;
// with 64 MB 17 us instead of 15.  (Its backward pass: 0 to 3 % either way, left alone.)
static bool ex_whole_lines(const ExpertRowArgs& a, int type) { return ex_row_bytes(a, type) % 128 == 0 && (uintptr_t)a.out % 128 == 0; }
static long long ex_bytes(const ExpertRowArgs& a, int type) { return (long long)a.n * a.k * ex_row_bytes(a, type); }

template <int T, int P, int PAST> static int ex_dispatch(ExpertRowArgs a, hipStream_t st) {
    const ExForm f = ex_form(a, T, 4);
    const unsigned grid = ex_grid((long long)a.n * a.tiles, f.group);
    if (!grid) return -1;
    if constexpr (P == 16) {
        if (f.u == 4) { MNE_LAUNCH((expert_dispatch_kernel<T, P, 4, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if (f.u == 3) { MNE_LAUNCH((expert_dispatch_kernel<T, P, 3, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if (f.u == 2) { MNE_LAUNCH((expert_dispatch_kernel<T, P, 2, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
    }
    MNE_LAUNCH((expert_dispatch_kernel<T, P, 1, PAST>), grid, EX_THREADS, 0, st, a, f.group);
    return 0;
}
template <int T, int P, int PAST> static int ex_combine(ExpertRowArgs a, hipStream_t st) {
    const ExForm f = ex_form(a, T, 4);
    const unsigned grid = ex_grid((long long)a.n * a.tiles, f.group);
    if (!grid) return -1;
    if constexpr (P == 16) {
        if (f.u == 4) { MNE_LAUNCH((expert_combine_kernel<T, P, 4, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if (f.u == 3) { MNE_LAUNCH((expert_combine_kernel<T, P, 3, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if (f.u == 2) { MNE_LAUNCH((expert_combine_kernel<T, P, 2, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
    }
    MNE_LAUNCH((expert_combine_kernel<T, P, 1, PAST>), grid, EX_THREADS, 0, st, a, f.group);
    return 0;
}
// (four rows at a time from three choices on)
template <int T, int P, int PAST, int K, int MOST> static int ex_backward(ExpertRowArgs a, hipStream_t st) {
    const ExForm f = ex_form(a, T, MOST);
    const unsigned grid = ex_grid(a.n, f.group);
    if (!grid) return -1;
    if constexpr (P == 16) {
        if constexpr (MOST >= 4) if (f.u == 4) { MNE_LAUNCH((expert_combine_backward_kernel<T, P, K, 4, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if constexpr (MOST >= 3) if (f.u == 3) { MNE_LAUNCH((expert_combine_backward_kernel<T, P, K, 3, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
        if (f.u == 2) { MNE_LAUNCH((expert_combine_backward_kernel<T, P, K, 2, PAST>), grid, EX_THREADS, 0, st, a, f.group); return 0; }
    }
    MNE_LAUNCH((expert_combine_backward_kernel<T, P, K, 1, PAST>), grid, EX_THREADS, 0, st, a, f.group);
    return 0;
}
template <int T, int P, int PAST> static int ex_backward_by_k(const ExpertRowArgs& a, hipStream_t st) {
    return a.k == 1 ? ex_backward<T, P, PAST, 1, 4>(a, st) : a.k == 2 ? ex_backward<T, P, PAST, 2, 3>(a, st) : ex_backward<T, P, PAST, 4, 2>(a, st);
}

// F<T, P, PAST>::go by the row's piece; rows shorter than 16 bytes never go past the caches
template <template <int, int, int> class F, int T> static int ex_by_piece(const ExpertRowArgs& a, int past, hipStream_t st) {
    switch (ex_piece(a, T)) {
        case 16: return past == 2 ? F<T, 16, 2>::go(a, st) : past == 1 ? F<T, 16, 1>::go(a, st) : F<T, 16, 0>::go(a, st);
        case 8: return F<T, 8, 0>::go(a, st);
        case 4: return F<T, 4, 0>::go(a, st);
        default:
            if constexpr (T != MNE_T_F32) return F<T, 2, 0>::go(a, st);
            else return -1;
    }
}
template <int T, int P, int PAST> struct ExDispatch {
    static int go(const ExpertRowArgs& a, hipStream_t st) { return ex_dispatch<T, P, PAST == 2 ? 1 : PAST>(a, st); }
};
template <int T, int P, int PAST> struct ExCombine {
    static int go(const ExpertRowArgs& a, hipStream_t st) { return ex_combine<T, P, PAST>(a, st); }
};
template <int T, int P, int PAST> struct ExBackward {
    static int go(const ExpertRowArgs& a, hipStream_t st) { return ex_backward_by_k<T, P, PAST == 2 ? 1 : PAST>(a, st); }
};
template <template <int, int, int> class F> static int ex_by_type(const ExpertRowArgs& a, int type, int past, hipStream_t st) {
    return type == MNE_T_F32 ? ex_by_piece<F, MNE_T_F32>(a, past, st) : type == MNE_T_BF16 ? ex_by_piece<F, MNE_T_BF16>(a, past, st) : ex_by_piece<F, MNE_T_F16>(a, past, st);
}

int mne_launch_expert_dispatch(ExpertRowArgs a, int type, hipStream_t st) {
    const int past = ex_whole_lines(a, type) && ex_bytes(a, type) < 1ll << 30;
    return type == MNE_T_F32 ? ex_by_piece<ExDispatch, MNE_T_F32>(a, past, st) : ex_by_piece<ExDispatch, MNE_T_F16>(a, past, st);   // (rows are copied: any 16-bit type)
}
int mne_launch_expert_combine(ExpertRowArgs a, int type, hipStream_t st) {
    return ex_by_type<ExCombine>(a, type, !ex_whole_lines(a, type) ? 0 : ex_bytes(a, type) < 1ll << 27 ? 1 : 2, st);
}
int mne_launch_expert_combine_backward(ExpertRowArgs a, int type, hipStream_t st) {
    return ex_by_type<ExBackward>(a, type, ex_whole_lines(a, type), st);
}
