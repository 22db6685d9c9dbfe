// routing.hip -- tokens (points, samples) sorted by expert, dealt to the experts' rows, and blended back with weights.
//
//   slot n k_max + k holds the expert ids[n][k] of token n; ids outside 0 .. experts - 1 name no expert
//   sort      a stable counting sort of the slots by expert: order[row] = slot, position[slot] = row, offsets[e] = first row of expert e
//   dispatch  out[position[n][k]] = x[n]                                  dx[n] = sum_k dout[position[n][k]]      (combine, no weights)
//   combine   out[n] = sum_k w[n][k] y[position[n][k]]                    dy[position[n][k]] = w[n][k] dout[n],  dw[n][k] = <dout[n], y[position[n][k]]>
//
// A row of the sorted side belongs to one slot, so nothing is added up across workgroups: no atomics on results, and the same bits
// every time.  Sums are fp32 over k = 0, 1, ... (and over a row in a fixed order); a 16-bit result is rounded to nearest even once.
#include "mne_device.h"
#include "mne_elem.h"
#include "mne_launch.h"

#define EX_THREADS 256
#define EX_WAVES (EX_THREADS / 64)
#define EX_CHUNK 4096                               // slots of a workgroup of the long form
#define EX_SHORT 16384                              // slots up to which one workgroup of 1024 does it all
#define EX_SHORT_EXPERTS 2000                       // its counters of 16 waves fit the LDS

// ---- sort ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int ex_id(const ExpertSortArgs& a, int slot) {        // what names no expert sorts behind all of them
    const long long e = a.wide ? ((const long long*)a.ids)[slot] : ((const int*)a.ids)[slot];
    return e >= 0 && e < a.experts ? (int)e : a.experts;
}

__global__ __launch_bounds__(EX_THREADS) void expert_count_kernel(ExpertSortArgs a) {
    MNE_DYN_LDS(lds);
    int* cnt = (int*)lds;
    for (int e = threadIdx.x; e <= a.experts; e += EX_THREADS) cnt[e] = 0;
    __syncthreads();
    const int first = (int)blockIdx.x * EX_CHUNK;
    for (int j = threadIdx.x; j < EX_CHUNK && first + j < a.m; j += EX_THREADS) atomicAdd(&cnt[ex_id(a, first + j)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += EX_THREADS) a.count[(long long)blockIdx.x * (a.experts + 1) + e] = cnt[e];
}

// count[chunk][e] becomes the number of e's slots in the chunks before, total[e] the number in all: 64 experts a workgroup, a
// quarter of the chunks a wave
__global__ __launch_bounds__(EX_THREADS) void expert_scan_kernel(ExpertSortArgs a) {
    __shared__ int part[EX_WAVES][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = (int)blockIdx.x * 64 + lane, stride = a.experts + 1;
    const int each = (a.chunks + EX_WAVES - 1) / EX_WAVES, lo = w * each, hi = lo + each < a.chunks ? lo + each : a.chunks;
    int sum = 0;
    if (e <= a.experts)
        for (int c = lo; c < hi; ++c) sum += a.count[(long long)c * stride + e];
    part[w][lane] = sum;
    __syncthreads();
    int run = 0, all = 0;
    for (int i = 0; i < EX_WAVES; ++i) {
        if (i < w) run += part[i][lane];
        all += part[i][lane];
    }
    if (e <= a.experts) {
        for (int c = lo; c < hi; ++c) {
            int* q = &a.count[(long long)c * stride + e];
            const int x = *q;
            *q = run;
            run += x;
        }
        if (w == 0) a.total[e] = all;
    }
}

// Rows of a workgroup's slots: WAVES waves of a.per_wave consecutive slots.  ALONE: one workgroup has all slots.
template <int WAVES, bool ALONE>
__global__ __launch_bounds__(WAVES * 64) void expert_place_kernel(ExpertSortArgs a) {
    MNE_DYN_LDS(lds);
    int* cnt = (int*)lds;                           // [WAVES][experts + 1]: counters, then next rows
    __shared__ int part[WAVES];
    const int bins = a.experts + 1, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int* mine = cnt + w * bins;
    for (int e = threadIdx.x; e < WAVES * bins; e += WAVES * 64) cnt[e] = 0;
    __syncthreads();
    const long long first = ((long long)blockIdx.x * WAVES + w) * a.per_wave;
    const int n = first < a.m ? (int)(a.m - first < a.per_wave ? a.m - first : a.per_wave) : 0;
    for (int j = lane; j < n; j += 64) atomicAdd(&mine[ex_id(a, (int)first + j)], 1);
    __syncthreads();
    // first row of every expert: a thread has a run of them, the threads' sums are scanned
    const int each = (bins + WAVES * 64 - 1) / (WAVES * 64), lo = threadIdx.x * each, hi = lo + each < bins ? lo + each : bins;
    int sum = 0;
    for (int e = lo; e < hi; ++e) {
        int t = 0;
        if (ALONE) for (int i = 0; i < WAVES; ++i) t += cnt[i * bins + e];
        else t = a.total[e];
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
        int t = 0, next = ALONE ? row : row + a.count[(long long)blockIdx.x * bins + e];
        for (int i = 0; i < WAVES; ++i) {
            const int c = cnt[i * bins + e];
            cnt[i * bins + e] = next;
            next += c;
            t += c;
        }
        row += ALONE ? t : a.total[e];
    }
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < bins) ++bits;
    for (int j0 = 0; j0 < n; j0 += 64) {            // 64 slots at a time, in order
        const int slot = (int)first + j0 + lane, live = j0 + lane < n, e = live ? ex_id(a, slot) : a.experts;
        unsigned long long peers = __ballot(live);  // the lanes with the same expert
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot((e >> b) & 1);
            peers &= (e >> b) & 1 ? set : ~set;
        }
        const int before = __popcll(peers & ((1ull << lane) - 1ull)), all = __popcll(peers);
        const int start = mine[e];
        MNE_WAVE_SYNC();
        if (live) {
            const int r = start + before;
            if (before == all - 1) mine[e] = r + 1;
            const bool named = e < a.experts;
            a.position[slot] = named ? r : -1;
            a.order[r] = named ? slot : -1;
        }
        MNE_WAVE_SYNC();
    }
}

static int ex_chunks(long long m) { return (int)((m + EX_CHUNK - 1) / EX_CHUNK); }
static bool ex_short(long long m, int experts) { return m <= EX_SHORT && experts <= EX_SHORT_EXPERTS; }

long long mne_expert_workspace_ints(long long m, int experts) {
    return ex_short(m, experts) ? 0 : ((long long)ex_chunks(m) + 1) * (experts + 1);
}

int mne_launch_expert_sort(ExpertSortArgs a, void* workspace, hipStream_t st) {
    const int bins = a.experts + 1;
    if (ex_short(a.m, a.experts)) {
        a.per_wave = (int)(((a.m + 15) / 16 + 63) / 64 * 64);
        const size_t lds = (size_t)16 * bins * sizeof(int);
        MNE_SET_MAX_LDS((expert_place_kernel<16, true>), lds);
        MNE_LAUNCH((expert_place_kernel<16, true>), 1, 1024, lds, st, a);
        return 0;
    }
    a.chunks = ex_chunks(a.m);
    a.per_wave = EX_CHUNK / EX_WAVES;
    a.count = (int*)workspace;
    a.total = a.count + (long long)a.chunks * bins;
    MNE_LAUNCH(expert_count_kernel, a.chunks, EX_THREADS, bins * sizeof(int), st, a);
    MNE_LAUNCH(expert_scan_kernel, (bins + 63) / 64, EX_THREADS, 0, st, a);
    const size_t lds = (size_t)EX_WAVES * bins * sizeof(int);
    MNE_SET_MAX_LDS((expert_place_kernel<EX_WAVES, false>), lds);
    MNE_LAUNCH((expert_place_kernel<EX_WAVES, false>), a.chunks, EX_THREADS, lds, st, a);
    return 0;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// A row is cut into 16-byte pieces and, behind them, single elements; column c of a row is piece c or element c - pieces.  The pieces
// are loaded and stored whole whatever the row's alignment is (element by element, odd widths would take eight times the instructions).
typedef unsigned ex_words __attribute__((ext_vector_type(4)));
typedef unsigned ex_words_in_memory __attribute__((ext_vector_type(4), aligned(2)));
template <int T> struct ExCol {
    typedef typename MneElem<T>::mem mem;
    static constexpr int N = 16 / (int)sizeof(mem);
    ex_words v;
    __device__ __forceinline__ void clear() { v = (ex_words)(0u); }
    __device__ __forceinline__ void load(const void* row, int c, int width) {
        const int pieces = width / N;
        if (c < pieces) v = ((const ex_words_in_memory*)row)[c];
        else {
            const mem* q = (const mem*)row + pieces * N + (c - pieces);
            clear();
            v.x = sizeof(mem) == 2 ? (unsigned)*(const unsigned short*)q : *(const unsigned*)q;
        }
    }
    __device__ __forceinline__ void store(void* row, int c, int width) const {
        const int pieces = width / N;
        if (c < pieces) ((ex_words_in_memory*)row)[c] = v;
        else {
            mem* q = (mem*)row + pieces * N + (c - pieces);
            if (sizeof(mem) == 2) *(unsigned short*)q = (unsigned short)v.x;
            else *(unsigned*)q = v.x;
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if (sizeof(mem) == 4) return __uint_as_float(v[j]);
        return MneElem<T>::get(__builtin_bit_cast(mem, (typename MneWord<sizeof(mem)>::type)(v[j >> 1] >> (j & 1 ? 16 : 0))));
    }
    __device__ __forceinline__ void put(const float* x) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (sizeof(mem) == 4) v[j] = __float_as_uint(x[j]);
            else {
                typedef typename MneWord<sizeof(mem)>::type word;
                v[j] = (unsigned)__builtin_bit_cast(word, MneElem<T>::put(x[N / 4 * j])) | (unsigned)__builtin_bit_cast(word, MneElem<T>::put(x[N / 4 * j + N / 4 - 1])) << 16;
            }
        }
    }
};

// GROUP lanes have a token and a tile of GROUP * U columns.
template <int T, int U>
__global__ __launch_bounds__(EX_THREADS) void expert_dispatch_kernel(ExpertRowArgs a, int group) {
    const long long unit = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    if (unit >= (long long)a.n * a.tiles) return;
    const int n = (int)(unit / a.tiles), c0 = (int)(unit % a.tiles) * group * U + l;
    const long long size = (long long)a.width * sizeof(typename MneElem<T>::mem), slot = (long long)n * a.k;
    const int total = *a.total;
    ExCol<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (c0 + u * group < a.cols) x[u].load((const char*)a.a + n * a.a_stride, c0 + u * group, a.width);
    for (int k = 0; k < a.k; ++k) {
        const int row = a.position[slot + k];
        if (row >= 0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * group < a.cols) x[u].store((char*)a.out + row * size, c0 + u * group, a.width);
        }
        if (slot + k >= total) {                    // a row behind the live ones: zero
            ExCol<T> zero;
            zero.clear();
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * group < a.cols) zero.store((char*)a.out + (slot + k) * size, c0 + u * group, a.width);
        }
    }
}

template <int T, int U, bool WEIGHTS>
__global__ __launch_bounds__(EX_THREADS) void expert_combine_kernel(ExpertRowArgs a, int group) {
    typedef ExCol<T> Col;
    const long long unit = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    if (unit >= (long long)a.n * a.tiles) return;
    const int n = (int)(unit / a.tiles), c0 = (int)(unit % a.tiles) * group * U + l;
    const long long size = (long long)a.width * sizeof(typename Col::mem), slot = (long long)n * a.k;
    float acc[U][Col::N] = {};
    for (int k = 0; k < a.k; ++k) {
        const int row = a.position[slot + k];
        if (row < 0) continue;
        const float w = WEIGHTS ? a.weights[slot + k] : 1.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * group < a.cols) {
                Col y;
                y.load((const char*)a.a + row * a.a_stride, c0 + u * group, a.width);
#pragma unroll
                for (int j = 0; j < Col::N; ++j) acc[u][j] = WEIGHTS ? fmaf(w, y.get(j), acc[u][j]) : acc[u][j] + y.get(j);
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

// GROUP lanes have a token: its row of dout against its rows of y, K slots at a time.
template <int T, int K>
__global__ __launch_bounds__(EX_THREADS) void expert_combine_backward_kernel(ExpertRowArgs a, int group) {
    typedef ExCol<T> Col;
    const long long n = ((long long)blockIdx.x * EX_THREADS + threadIdx.x) / group;
    const int l = threadIdx.x & (group - 1);
    const bool there = n < a.n;                     // (all lanes stay: they add up the dot products together)
    const long long size = (long long)a.width * sizeof(typename Col::mem), slot = n * a.k;
    const int total = *a.total;
    for (int k0 = 0; k0 < a.k; k0 += K) {
        int row[K];
        float w[K], dot[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool on = there && k0 + i < a.k;
            row[i] = on ? a.position[slot + k0 + i] : -1;
            w[i] = on && a.weights ? a.weights[slot + k0 + i] : 1.0f;
            dot[i] = 0.0f;
        }
        if (there)
            for (int c = l; c < a.cols; c += group) {
                Col d;
                d.load((const char*)a.a + n * a.a_stride, c, a.width);
                const int live = c < a.width / Col::N ? Col::N : 1;
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    if (k0 + i >= a.k) continue;
                    if (row[i] >= 0) {
                        if (a.dw) {
                            Col y;
                            y.load((const char*)a.b + row[i] * a.b_stride, c, a.width);
#pragma unroll
                            for (int j = 0; j < Col::N; ++j)
                                if (j < live) dot[i] = fmaf(d.get(j), y.get(j), dot[i]);
                        }
                        if (a.out) {
                            Col o;
                            float x[Col::N];
#pragma unroll
                            for (int j = 0; j < Col::N; ++j) x[j] = w[i] * d.get(j);
                            o.put(x);
                            o.store((char*)a.out + row[i] * size, c, a.width);
                        }
                    }
                    if (a.out && slot + k0 + i >= total) {
                        Col zero;
                        zero.clear();
                        zero.store((char*)a.out + (slot + k0 + i) * size, c, a.width);
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

// columns of a row, and the lanes that take one: a power of two, at most a wave
static int ex_columns(ExpertRowArgs& a, int type) {
    const int per = type == MNE_T_F32 ? 4 : 8;
    a.cols = a.width / per + a.width % per;
    int group = 1;
    while (group < a.cols && group < 64) group <<= 1;
    return group;
}
static unsigned ex_grid(long long units, int group) { return (unsigned)((units * group + EX_THREADS - 1) / EX_THREADS); }

template <int T> static void ex_dispatch(ExpertRowArgs a, hipStream_t st) {
    const int group = ex_columns(a, T), u = a.cols > 128 ? 4 : a.cols > 64 ? 2 : 1;
    a.tiles = (a.cols + group * u - 1) / (group * u);
    const unsigned grid = ex_grid((long long)a.n * a.tiles, group);
    if (u == 4) MNE_LAUNCH((expert_dispatch_kernel<T, 4>), grid, EX_THREADS, 0, st, a, group);
    else if (u == 2) MNE_LAUNCH((expert_dispatch_kernel<T, 2>), grid, EX_THREADS, 0, st, a, group);
    else MNE_LAUNCH((expert_dispatch_kernel<T, 1>), grid, EX_THREADS, 0, st, a, group);
}
template <int T, bool W> static void ex_combine(ExpertRowArgs a, hipStream_t st) {
    const int group = ex_columns(a, T), u = a.cols > 64 ? 2 : 1;
    a.tiles = (a.cols + group * u - 1) / (group * u);
    const unsigned grid = ex_grid((long long)a.n * a.tiles, group);
    if (u == 2) MNE_LAUNCH((expert_combine_kernel<T, 2, W>), grid, EX_THREADS, 0, st, a, group);
    else MNE_LAUNCH((expert_combine_kernel<T, 1, W>), grid, EX_THREADS, 0, st, a, group);
}
template <int T> static void ex_backward(ExpertRowArgs a, hipStream_t st) {
    const int group = ex_columns(a, T);
    const unsigned grid = ex_grid(a.n, group);
    if (a.k == 1) MNE_LAUNCH((expert_combine_backward_kernel<T, 1>), grid, EX_THREADS, 0, st, a, group);
    else if (a.k == 2) MNE_LAUNCH((expert_combine_backward_kernel<T, 2>), grid, EX_THREADS, 0, st, a, group);
    else MNE_LAUNCH((expert_combine_backward_kernel<T, 4>), grid, EX_THREADS, 0, st, a, group);
}

int mne_launch_expert_dispatch(ExpertRowArgs a, int type, hipStream_t st) {
    if (type == MNE_T_F32) ex_dispatch<MNE_T_F32>(a, st);
    else ex_dispatch<MNE_T_F16>(a, st);             // (rows are copied: any 16-bit type)
    return 0;
}
int mne_launch_expert_combine(ExpertRowArgs a, int type, hipStream_t st) {
    if (type == MNE_T_F32) a.weights ? ex_combine<MNE_T_F32, true>(a, st) : ex_combine<MNE_T_F32, false>(a, st);
    else if (type == MNE_T_BF16) a.weights ? ex_combine<MNE_T_BF16, true>(a, st) : ex_combine<MNE_T_BF16, false>(a, st);
    else a.weights ? ex_combine<MNE_T_F16, true>(a, st) : ex_combine<MNE_T_F16, false>(a, st);
    return 0;
}
int mne_launch_expert_combine_backward(ExpertRowArgs a, int type, hipStream_t st) {
    if (type == MNE_T_F32) ex_backward<MNE_T_F32>(a, st);
    else if (type == MNE_T_BF16) ex_backward<MNE_T_BF16>(a, st);
    else ex_backward<MNE_T_F16>(a, st);
    return 0;
}
