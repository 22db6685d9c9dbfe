// adamw.hip -- one AdamW step (decoupled weight decay) over many tensors in one launch, moments in 32 bits or in 8.
//
//   p = p * (1 - lr wd);  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
//   p = p - step_size * (m / (sqrt(v) / root_bc2 + eps)),   step_size = lr / (1 - b1^t),  root_bc2 = sqrt(1 - b2^t)
//
// The arithmetic is fp32 whatever the types in memory are (parameters and gradients: fp32, bf16, fp16); a 16-bit parameter is
// rounded to nearest even once, when it is stored.
//
// 8-bit moments: a tensor's memory is cut into blocks of 256 elements, each with two fp32 scales.
//   m       = sign(c) c^2 * scale_m,  c int8 in -127..127,  scale_m = max |m| / 127^2
//   sqrt(v) = c^2 * scale_r,          c uint8 in 0..255,    scale_r = max sqrt(v) / 255^2
// Codes on a square-law scale: next to the block's largest value one code is 1.6 % (m) / 0.8 % (sqrt v), at a hundredth of it 16 % /
// 8 %, and the range reaches down to 6e-5 / 1.5e-5 of it.  With x = |m| 127^2 / max the code is floor(sqrt x), or one more with the
// probability that makes its square right on average: u (2 c + 1) < x - c^2, u a dither of 16 bits.  Rounding to the nearest code
// instead would hold a moment still that changes by less than half a code a step (b2 = 0.999 moves sqrt(v) by 0.05 %).
// sqrt(v) > 0 keeps a code of at least 1: an update is never divided by eps alone because a small moment was rounded away.
// A block in which a new moment is not finite holds NaN from then on (scales NaN, codes 0): all 256 elements share the scale that would
// have to be infinite.  A gradient does that which is not finite itself, and one of 1.85e19 and more, whose square is infinite in fp32
// (32-bit moments keep the infinity to that one element, and its parameter stands still).
// What enters the codes is plain IEEE fp32 in the order written here (the build forbids contraction), so the codes do not depend on
// the launch or on the machine.
//
// With 32-bit moments the step is bound by memory: 38.4 M fp32 values 180 us (28 bytes each, 6.0 TB/s), 67 M bf16 values in 256 tensors 250 us
// (22 bytes, 5.9 TB/s).  With 8-bit ones it is where the parameters are fp32 (38.4 M: 96 us, 16 bytes, 6.4 TB/s); with bf16 parameters (10
// bytes) it is bound by its 83 vector instructions an element, four of them roots and reciprocals: 67 M values 169 us (4.0 TB/s).
#include "mne_device.h"
#include "mne_elem.h"
#include "mne_launch.h"

#define AW_THREADS 256
#define AW_BLOCK 256                                 // elements that share two scales
// Elements a workgroup takes: 4 a thread with 32-bit moments, and 8 a thread (32 lanes a block) with 8-bit ones.  Measured: 32-bit
// moments, 67 M bf16 values in 256 tensors: 250 us with 4 a thread, 291 with 8, 331 with 16 (38.4 M fp32 values: 180, 186, 183); 8-bit
// moments: 187 us with 32 lanes a block, 204 with 16, 216 with 64, which are 0.5 us faster than 32 in the smallest calls (5.7 us).  (All
// of these before the last 5 %, which came to each of them.)
#define AW_PAST (1ll << 29)                          // bytes of a call from which on it goes past the caches
#define AW_EACH32 4
#define AW_LANES8 32
#define AW_WG32 (AW_THREADS * AW_EACH32)
#define AW_WG8 (AW_THREADS / AW_LANES8 * AW_BLOCK)

// a multiply-xorshift mix of 32 bits; shifts and factors are those of a published hash (C. Wellons, "Prospecting for hash functions", 2018)
__device__ __forceinline__ unsigned aw_mix(unsigned h) {
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
#define AW_GOLD 0x9E3779B1u

// the tensor that workgroup `blk` works on: first[s] <= blk < first[s + 1]
__device__ __forceinline__ int aw_segment(const int* first, int n, int blk) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= blk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// N consecutive elements of memory from (to) element i, as fp32: vectors of up to 16 bytes, or, with FULL false, element by element
// and only those below n (zeros stand for the others).
template <int T, int N, bool FULL, bool PAST>
__device__ __forceinline__ void aw_load(float* out, const void* base, long long i, long long n) {
    typedef typename MneElem<T>::mem mem;
    const mem* q = (const mem*)base + i;
    if (FULL) {
        constexpr int B = N * (int)sizeof(mem) < 16 ? N * (int)sizeof(mem) : 16;
        union { MneBytes<B> v[N * sizeof(mem) / B]; mem e[N]; } r;
#pragma unroll
        for (int k = 0; k < N * (int)sizeof(mem) / B; ++k) r.v[k] = PAST ? mne_load_once((const MneBytes<B>*)q + k) : ((const MneBytes<B>*)q)[k];
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = MneElem<T>::get(r.e[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = i + k < n ? MneElem<T>::get(q[k]) : 0.0f;
    }
}
template <int T, int N, bool FULL, bool PAST>
__device__ __forceinline__ void aw_store(const float* x, void* base, long long i, long long n) {
    typedef typename MneElem<T>::mem mem;
    mem* q = (mem*)base + i;
    if (FULL) {
        constexpr int B = N * (int)sizeof(mem) < 16 ? N * (int)sizeof(mem) : 16;
        union { MneBytes<B> v[N * sizeof(mem) / B]; mem e[N]; } r;
#pragma unroll
        for (int k = 0; k < N; ++k) r.e[k] = MneElem<T>::put(x[k]);
#pragma unroll
        for (int k = 0; k < N * (int)sizeof(mem) / B; ++k) {
            if (PAST) mne_store_once((MneBytes<B>*)q + k, r.v[k]);
            else ((MneBytes<B>*)q)[k] = r.v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) if (i + k < n) q[k] = MneElem<T>::put(x[k]);
    }
}

// Consecutive elements of a thread's pieces: 16 bytes of the parameter, as far as the thread has that many.
template <int PT, int EACH> struct AwPiece { static constexpr int N = PT == MNE_T_F32 || EACH < 8 ? 4 : 8; };

template <int PT, int GT, bool PAST, bool FULL>
__device__ __forceinline__ void adamw32_body(const Adamw32Args& a, const AdamwHyper& h, int s, long long base) {
    constexpr int N = AwPiece<PT, AW_EACH32>::N, K = AW_EACH32 / N;
    const long long n = a.n[s], i0 = base + threadIdx.x * N;
    float p[K][N], g[K][N], m[K][N], v[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = i0 + k * (AW_THREADS * N);
        aw_load<PT, N, FULL, PAST>(p[k], a.p[s], i, n);
        aw_load<GT, N, FULL, PAST>(g[k], a.g[s], i, n);
        aw_load<MNE_T_F32, N, FULL, PAST>(m[k], a.m[s], i, n);
        aw_load<MNE_T_F32, N, FULL, PAST>(v[k], a.v[s], i, n);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = i0 + k * (AW_THREADS * N);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            m[k][j] = m[k][j] * h.b1 + g[k][j] * h.omb1;
            v[k][j] = v[k][j] * h.b2 + (g[k][j] * g[k][j]) * h.omb2;
            p[k][j] = p[k][j] * h.decay - h.step_size * (m[k][j] / (sqrtf(v[k][j]) / h.root_bc2 + h.eps));
            g[k][j] = 0.0f;
        }
        aw_store<PT, N, FULL, PAST>(p[k], a.p[s], i, n);
        aw_store<MNE_T_F32, N, FULL, PAST>(m[k], a.m[s], i, n);
        aw_store<MNE_T_F32, N, FULL, PAST>(v[k], a.v[s], i, n);
        if (a.zero_grad) aw_store<GT, N, FULL, PAST>(g[k], a.g[s], i, n);
    }
}

template <int PT, int GT, bool PAST>
__global__ __launch_bounds__(AW_THREADS) void adamw32_kernel(Adamw32Args a) {
    const int s = aw_segment(a.first, a.n_seg, (int)blockIdx.x);
    AdamwHyper h = a.h;
    if (a.clk.bias_table) clock_bias(a.clk, h.lr, h.step, h.step_size, h.root_bc2);
    const long long base = (long long)((int)blockIdx.x - a.first[s]) * AW_WG32;
    if (base + AW_WG32 <= a.n[s]) adamw32_body<PT, GT, PAST, true>(a, h, s, base);
    else adamw32_body<PT, GT, PAST, false>(a, h, s, base);
}

// Code of x in 0..most^2 with the dither k / 65536: floor of the root, or one more if k / 65536 (2 c + 1) < x - c^2.  The floor is exact
// with a root that is 1 ulp off: it is the floor of the root of floor(x) + 1/2, which is no nearer than 1 / (4 most) to a whole number.
// The difference is exact too (c^2 is, and it is a multiple of x's last place, no larger than x).
// SOME: what is not zero gets at least 1 (below 1 the step to it is taken whatever the dither is: its weight, 2 c + 1, is held to c).
template <bool SOME> __device__ __forceinline__ int aw_code(float x, unsigned short k) {
    const int c = (int)mne_sqrt_fast(floorf(x) + 0.5f);
    const float f = (float)c, w = fmaf(f, 2.0f / 65536.0f, 1.0f / 65536.0f);
    return (float)k * (SOME ? fminf(w, f) : w) < fmaf(-f, f, x) ? c + 1 : c;
}

__device__ __forceinline__ unsigned aw_max(unsigned x) {        // over the lanes of a block
    x = mne_max16(x);
#pragma unroll
    for (int d = 16; d < AW_LANES8; d <<= 1) {
        const unsigned o = __shfl_xor(x, d);
        x = o > x ? o : x;
    }
    return x;
}

// LANES lanes have a block of 256 elements, EACH of them each.
template <int PT, int GT, bool PAST, bool FULL>
__device__ __forceinline__ void adamw8_body(const Adamw8Args& a, const AdamwHyper& h, int step, int s, long long b) {
    constexpr int LANES = AW_LANES8, EACH = AW_BLOCK / LANES, N = AwPiece<PT, EACH>::N, K = EACH / N;
    const int l = threadIdx.x % LANES;
    const long long n = a.n[s], i0 = b * AW_BLOCK + l * N;
    const bool there = FULL || b * AW_BLOCK < n;
    const float2 scale = there ? ((const float2*)a.scales[s])[b] : make_float2(0.0f, 0.0f);
    float m[K][N], r[K][N];
    {
        float p[K][N], g[K][N];
        union { MneBytes<N> v; signed char c[N]; } mc[K];
        union { MneBytes<N> v; unsigned char c[N]; } rc[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const long long i = i0 + k * (LANES * N);
            aw_load<PT, N, FULL, PAST>(p[k], a.p[s], i, n);
            aw_load<GT, N, FULL, PAST>(g[k], a.g[s], i, n);
            if (FULL) {
                mc[k].v = *(const MneBytes<N>*)((const signed char*)a.m[s] + i);
                rc[k].v = *(const MneBytes<N>*)((const unsigned char*)a.v[s] + i);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    mc[k].c[j] = i + j < n ? ((const signed char*)a.m[s])[i + j] : (signed char)0;
                    rc[k].c[j] = i + j < n ? ((const unsigned char*)a.v[s])[i + j] : (unsigned char)0;
                }
            }
        }
        unsigned least = 0xFFFFFFFFu;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float c = (float)mc[k].c[j], d = (float)rc[k].c[j], gg = g[k][j], r0 = d * d * scale.y;
                m[k][j] = (c * fabsf(c) * scale.x) * h.b1 + gg * h.omb1;
                r[k][j] = (r0 * r0) * h.b2 + (gg * gg) * h.omb2;
                const unsigned below = __float_as_uint(r[k][j]) - 1u;            // zero is out of the way, at the top
                least = below < least ? below : least;
            }
        if (least < 0x0F800000u - 1u) {               // a square below 2^-96: the root with scaling
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) r[k][j] = sqrtf(r[k][j]);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) r[k][j] = mne_sqrt_rn(r[k][j]);
        }
        // The quotient: a reciprocal 1 ulp off, and for a 32-bit parameter one correction, which leaves a rounded quotient (a 16-bit one is
        // rounded at 2^-9 or 2^-12 anyway, and its step is bound by instructions).  The reciprocal takes a number below 2^-126, which eps may
        // be where there has been no gradient, for zero: the quotient is formed 2^24 too small.
        const float up = 16777216.0f, inv = up / h.root_bc2, eps = up * h.eps, size = up * h.step_size;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const long long i = i0 + k * (LANES * N);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = fmaf(r[k][j], inv, eps), y = mne_rcp_fast(d);
                float q = m[k][j] * y;
                if (PT == MNE_T_F32) {
                    const float off = fmaf(-d, q, m[k][j]);
                    q = off == off ? fmaf(off, y, q) : q;          // (not where d is infinite: the quotient is 0)
                }
                p[k][j] = fmaf(-size, q, p[k][j] * h.decay);
                g[k][j] = 0.0f;
            }
            aw_store<PT, N, FULL, PAST>(p[k], a.p[s], i, n);
            if (a.zero_grad) aw_store<GT, N, FULL, PAST>(g[k], a.g[s], i, n);
        }
    }
    // Largest magnitudes of the block.  Of sqrt(v) by the bits, where NaN is above infinity; where all of it is finite and the block's m
    // was, all of m is (a gradient that is not finite, or too large for m, is too large for sqrt(v)).
    float most = 0.0f;
    unsigned br = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const unsigned ur = __float_as_uint(r[k][j]);
            most = fmaxf(most, fabsf(m[k][j]));
            br = ur > br ? ur : br;
        }
    unsigned bm = __float_as_uint(most);
    br = aw_max(br);
    if (__ballot(br >= 0x7F800000u || !(fabsf(scale.x) < __uint_as_float(0x7F800000u)))) {      // (the whole wave goes this way)
        bm = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned um = __float_as_uint(m[k][j]) & 0x7FFFFFFFu;
                bm = um > bm ? um : bm;
            }
    }
    bm = aw_max(bm);
    const bool fine_m = bm < 0x7F800000u, fine_r = br < 0x7F800000u;
    const float fm = __uint_as_float(bm), fr = __uint_as_float(br);
    const bool some_m = fine_m && fm > 7.8886090522101181e-31f, some_r = fine_r && fr > 0.0f;      // 2^-100: 127^2 / max stays finite
    // Four quotients a block, one for each lane of four: 127^2 / max |m|, 255^2 / max sqrt(v), and the scales the other way round.
    const int q = l & 3;
    const float top = q & 1 ? 65025.0f : 16129.0f, big = q & 1 ? fr : fm, quotient = q & 2 ? big / top : top / big;
    const float up_m = mne_quad(quotient, 0), up_r = mne_quad(quotient, 1), scale_m = mne_quad(quotient, 2), scale_r = mne_quad(quotient, 3);
    const float im = some_m ? up_m : 0.0f, ir = some_r ? up_r : 0.0f;
    if (!(fine_m && fine_r)) {                        // codes 0 in what is not finite
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (!fine_m) m[k][j] = 0.0f;
                if (!fine_r) r[k][j] = 0.0f;
            }
    }
    // (the blocks of a wave one after the other: their numbers are the wave's, so the scalar unit does this)
    const unsigned key = a.key[s] + (unsigned)step * AW_GOLD, b0 = (unsigned)mne_first_lane((int)b);
    unsigned kb = aw_mix(key ^ aw_mix(b0));
#pragma unroll
    for (int k = 1; k < 64 / LANES; ++k) {
        const unsigned other = aw_mix(key ^ aw_mix(b0 + (unsigned)k));
        kb = (threadIdx.x & 63) / LANES == k ? other : kb;
    }
    kb += (unsigned)(l * N) * AW_GOLD;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = i0 + k * (LANES * N);
        unsigned cm[N], cr[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            unsigned u = kb + (unsigned)(k * LANES * N + j) * AW_GOLD;
            u = (u ^ (u >> 16)) * 0x7FEB352Du;
            u ^= u >> 15;
            int x = aw_code<false>(fabsf(m[k][j]) * im, (unsigned short)u);
            x = x < 127 ? x : 127;
            cm[j] = (unsigned)(m[k][j] < 0.0f ? -x : x);
            x = aw_code<true>(r[k][j] * ir, (unsigned short)(u >> 16));
            cr[j] = (unsigned)(x < 255 ? x : 255);
        }
        if (FULL) {
            union { MneBytes<N> v; unsigned w[N / 4]; } mc, rc;
#pragma unroll
            for (int j = 0; j < N / 4; ++j) {
                mc.w[j] = mne_pack4(cm[4 * j], cm[4 * j + 1], cm[4 * j + 2], cm[4 * j + 3]);
                rc.w[j] = mne_pack4(cr[4 * j], cr[4 * j + 1], cr[4 * j + 2], cr[4 * j + 3]);
            }
            *(MneBytes<N>*)((signed char*)a.m[s] + i) = mc.v;
            *(MneBytes<N>*)((unsigned char*)a.v[s] + i) = rc.v;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (i + j < n) { ((unsigned char*)a.m[s])[i + j] = (unsigned char)cm[j]; ((unsigned char*)a.v[s])[i + j] = (unsigned char)cr[j]; }
        }
    }
    if (l == 0 && there) {
        const float nan = __uint_as_float(0x7FC00000u);
        ((float2*)a.scales[s])[b] = make_float2(fine_m ? (some_m ? scale_m : 0.0f) : nan, fine_r ? (some_r ? scale_r : 0.0f) : nan);
    }
}

template <int PT, int GT, bool PAST>
__global__ __launch_bounds__(AW_THREADS) void adamw8_kernel(Adamw8Args a) {
    const int s = aw_segment(a.first, a.n_seg, (int)blockIdx.x);
    AdamwHyper h = a.h;
    int step = h.step;
    if (a.clk.bias_table) {
        clock_bias(a.clk, h.lr, h.step, h.step_size, h.root_bc2);
        step += *a.clk.step_offset;
    }
    constexpr int BLOCKS = AW_THREADS / AW_LANES8;
    const long long wg = (int)blockIdx.x - a.first[s], b = wg * BLOCKS + threadIdx.x / AW_LANES8;
    if ((wg + 1) * AW_WG8 <= a.n[s]) adamw8_body<PT, GT, PAST, true>(a, h, step, s, b);
    else adamw8_body<PT, GT, PAST, false>(a, h, step, s, b);
}

// What 8-bit moments stand for, in 32 bits: exp_avg and exp_avg_sq, four elements a thread.  Written past the caches at every size: 38.4 M
// values 54 us instead of 68, 134 M 188 instead of 222, 4.2 M 6.8 instead of 8.1, with an addition of both behind it 131 instead of 135, 481
// instead of 503 and 16.3 either way; up to 1 M values the launch is all there is.  (At 16.8 M alone the reader gains from the caches: 24.8
// and with it 57.1, against 25.7 and 54.4.)
__global__ __launch_bounds__(AW_THREADS) void adamw_moments_kernel(const signed char* mc, const unsigned char* rc, const float* scales,
                                                                   long long n, float* m, float* v) {
    const long long i = 4 * ((long long)blockIdx.x * AW_THREADS + threadIdx.x);
    if (i >= n) return;
    const float2 scale = ((const float2*)scales)[i / AW_BLOCK];
    union { MneBytes<4> v; signed char c[4]; } a;
    union { MneBytes<4> v; unsigned char c[4]; } b;
    const bool full = i + 4 <= n;
    if (full) {
        a.v = *(const MneBytes<4>*)(mc + i);
        b.v = *(const MneBytes<4>*)(rc + i);
    } else {
        for (int j = 0; j < 4; ++j) {
            a.c[j] = i + j < n ? mc[i + j] : (signed char)0;
            b.c[j] = i + j < n ? rc[i + j] : (unsigned char)0;
        }
    }
    float x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float c = (float)a.c[j], d = (float)b.c[j], r = d * d * scale.y;
        x[j] = c * fabsf(c) * scale.x;
        y[j] = r * r;
    }
    if (full) {
        aw_store<MNE_T_F32, 4, true, true>(x, m, i, n);
        aw_store<MNE_T_F32, 4, true, true>(y, v, i, n);
    } else {
        aw_store<MNE_T_F32, 4, false, false>(x, m, i, n);
        aw_store<MNE_T_F32, 4, false, false>(y, v, i, n);
    }
}

template <class Args, template <int, int> class Launch>
static int aw_by_type(const Args& a, int pt, int gt, unsigned blocks, bool past, hipStream_t st) {
    if (pt == MNE_T_F32 && gt == MNE_T_F32) Launch<MNE_T_F32, MNE_T_F32>::go(a, blocks, past, st);
    else if (pt == MNE_T_F32 && gt == MNE_T_BF16) Launch<MNE_T_F32, MNE_T_BF16>::go(a, blocks, past, st);
    else if (pt == MNE_T_F32 && gt == MNE_T_F16) Launch<MNE_T_F32, MNE_T_F16>::go(a, blocks, past, st);
    else if (pt == MNE_T_BF16 && gt == MNE_T_F32) Launch<MNE_T_BF16, MNE_T_F32>::go(a, blocks, past, st);
    else if (pt == MNE_T_BF16 && gt == MNE_T_BF16) Launch<MNE_T_BF16, MNE_T_BF16>::go(a, blocks, past, st);
    else if (pt == MNE_T_F16 && gt == MNE_T_F32) Launch<MNE_T_F16, MNE_T_F32>::go(a, blocks, past, st);
    else if (pt == MNE_T_F16 && gt == MNE_T_F16) Launch<MNE_T_F16, MNE_T_F16>::go(a, blocks, past, st);
    else return -1;
    return 0;
}
template <int PT, int GT> struct Launch32 {
    static void go(const Adamw32Args& a, unsigned blocks, bool past, hipStream_t st) {
        if (past) MNE_LAUNCH((adamw32_kernel<PT, GT, true>), blocks, AW_THREADS, 0, st, a);
        else MNE_LAUNCH((adamw32_kernel<PT, GT, false>), blocks, AW_THREADS, 0, st, a);
    }
};
template <int PT, int GT> struct Launch8 {
    static void go(const Adamw8Args& a, unsigned blocks, bool past, hipStream_t st) {
        if (past) MNE_LAUNCH((adamw8_kernel<PT, GT, true>), blocks, AW_THREADS, 0, st, a);
        else MNE_LAUNCH((adamw8_kernel<PT, GT, false>), blocks, AW_THREADS, 0, st, a);
    }
};

int mne_launch_adamw32(const Adamw32Args& a, int p_type, int g_type, unsigned blocks, bool past, hipStream_t st) {
    return aw_by_type<Adamw32Args, Launch32>(a, p_type, g_type, blocks, past, st);
}
int mne_launch_adamw8(const Adamw8Args& a, int p_type, int g_type, unsigned blocks, bool past, hipStream_t st) {
    return aw_by_type<Adamw8Args, Launch8>(a, p_type, g_type, blocks, past, st);
}
int mne_launch_adamw_moments(const signed char* mc, const unsigned char* rc, const float* scales, long long n, float* m, float* v, hipStream_t st) {
    MNE_LAUNCH(adamw_moments_kernel, (unsigned)((n + 4 * AW_THREADS - 1) / (4 * AW_THREADS)), AW_THREADS, 0, st, mc, rc, scales, n, m, v);
    return 0;
}
// Calls that touch more than twice what the last cache holds leave it to others: 33.6 M fp32 values (940 MB) 163 us instead of 181; of less,
// the next step finds a part there again -- 16.8 M values (470 MB) 69 us, and 79 past it.
bool mne_adamw_past(long long elements, int p_type, int g_type, int state_bits) {
    return elements * (2 * (p_type == MNE_T_F32 ? 4 : 2) + (g_type == MNE_T_F32 ? 4 : 2) + (state_bits == 8 ? 4 : 16)) > AW_PAST;
}
int mne_adamw_per_wg(int state_bits) { return state_bits == 8 ? AW_WG8 : AW_WG32; }
unsigned mne_adamw_key(unsigned seed, unsigned ordinal) {
    unsigned h = seed + ordinal * AW_GOLD;
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
