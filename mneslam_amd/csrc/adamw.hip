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
// A block that meets a value that is not finite holds NaN from then on (scales NaN, codes 0), as a 32-bit moment would.
// What enters the codes is plain IEEE fp32 in the order written here (the build forbids contraction), so the codes do not depend on
// the launch or on the machine.
#include "mne_device.h"
#include "mne_launch.h"

#define AW_THREADS 256
#define AW_BLOCK 256                                 // elements that share two scales
#define AW_PER_WG 4096                               // elements of a workgroup: 16 of each thread

__device__ __forceinline__ unsigned aw_mix(unsigned h) {      // a multiply-xorshift mix of 32 bits
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
#define AW_GOLD 0x9E3779B1u

template <int T> struct AwType;                      // how an element is held: MNE_T_F32 / _BF16 / _F16
template <> struct AwType<MNE_T_F32> {
    typedef float mem;
    static __device__ __forceinline__ float get(mem x) { return x; }
    static __device__ __forceinline__ mem put(float x) { return x; }
};
template <> struct AwType<MNE_T_BF16> {
    typedef unsigned short mem;
    static __device__ __forceinline__ float get(mem x) { return mne_bf16_to_float(x); }
    static __device__ __forceinline__ mem put(float x) { return mne_float_to_bf16(x); }
};
template <> struct AwType<MNE_T_F16> {
    typedef _Float16 mem;
    static __device__ __forceinline__ float get(mem x) { return (float)x; }
    static __device__ __forceinline__ mem put(float x) { return (_Float16)x; }
};

// the tensor that workgroup `blk` works on: first[s] <= blk < first[s + 1]
__device__ __forceinline__ int aw_segment(const int* first, int n, int blk) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= blk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int PT, int GT>
__global__ __launch_bounds__(AW_THREADS) void adamw32_kernel(Adamw32Args a) {
    const int s = aw_segment(a.first, a.n_seg, (int)blockIdx.x);
    AdamwHyper h = a.h;
    if (a.clk.bias_table) clock_bias(a.clk, h.lr, h.step, h.step_size, h.root_bc2);
    typename AwType<PT>::mem* p = (typename AwType<PT>::mem*)a.p[s];
    typename AwType<GT>::mem* g = (typename AwType<GT>::mem*)a.g[s];
    float *m = (float*)a.m[s], *v = (float*)a.v[s];
    const long long n = a.n[s], base = (long long)((int)blockIdx.x - a.first[s]) * AW_PER_WG;
    for (int k = 0; k < AW_PER_WG / AW_THREADS; ++k) {
        const long long i = base + k * AW_THREADS + threadIdx.x;
        if (i >= n) return;
        const float gg = AwType<GT>::get(g[i]);
        const float mm = m[i] * h.b1 + gg * h.omb1;
        const float vv = v[i] * h.b2 + (gg * gg) * h.omb2;
        p[i] = AwType<PT>::put(AwType<PT>::get(p[i]) * h.decay - h.step_size * (mm / (sqrtf(vv) / h.root_bc2 + h.eps)));
        m[i] = mm; v[i] = vv;
        if (a.zero_grad) g[i] = AwType<GT>::put(0.0f);
    }
}

// code of x in 0..top (top = most^2): floor of the root, or one more where the dither says so
__device__ __forceinline__ float aw_code(float x, float u) {
    float c = floorf(sqrtf(x));
    if (c * c > x) c -= 1.0f;                         // the root was rounded up to the next whole number
    return u * (2.0f * c + 1.0f) < x - c * c ? c + 1.0f : c;
}

template <int PT, int GT>
__global__ __launch_bounds__(AW_THREADS) void adamw8_kernel(Adamw8Args a) {
    const int s = aw_segment(a.first, a.n_seg, (int)blockIdx.x), lane = threadIdx.x & 63;
    AdamwHyper h = a.h;
    int step = h.step;
    if (a.clk.bias_table) {
        clock_bias(a.clk, h.lr, h.step, h.step_size, h.root_bc2);
        step += *a.clk.step_offset;
    }
    typename AwType<PT>::mem* p = (typename AwType<PT>::mem*)a.p[s];
    typename AwType<GT>::mem* g = (typename AwType<GT>::mem*)a.g[s];
    signed char* mc = (signed char*)a.m[s];
    unsigned char* rc = (unsigned char*)a.v[s];
    const long long n = a.n[s];
    for (int k = 0; k < 4; ++k) {                     // one wave a block of 256, four blocks a wave
        const long long b = (long long)((int)blockIdx.x - a.first[s]) * (AW_PER_WG / AW_BLOCK) + (threadIdx.x >> 6) * 4 + k;
        if (b * AW_BLOCK >= n) return;
        const float sm = a.scales[s][2 * b], sr = a.scales[s][2 * b + 1];
        float mm[4], rr[4];
        unsigned bm = 0, br = 0;
        for (int j = 0; j < 4; ++j) {
            const long long i = b * AW_BLOCK + j * 64 + lane;
            mm[j] = rr[j] = 0.0f;
            if (i < n) {
                const float gg = AwType<GT>::get(g[i]), c = (float)mc[i], d = (float)rc[i], r0 = d * d * sr;
                mm[j] = (c * fabsf(c) * sm) * h.b1 + gg * h.omb1;
                rr[j] = sqrtf((r0 * r0) * h.b2 + (gg * gg) * h.omb2);
                p[i] = AwType<PT>::put(AwType<PT>::get(p[i]) * h.decay - h.step_size * (mm[j] / (rr[j] / h.root_bc2 + h.eps)));
                if (a.zero_grad) g[i] = AwType<GT>::put(0.0f);
            }
            const unsigned um = __float_as_uint(mm[j]) & 0x7FFFFFFFu, ur = __float_as_uint(rr[j]) & 0x7FFFFFFFu;
            bm = um > bm ? um : bm;                   // order of the bits = order of the magnitudes, NaN above infinity
            br = ur > br ? ur : br;
        }
        for (int d = 32; d; d >>= 1) {
            const unsigned om = __shfl_xor(bm, d), orr = __shfl_xor(br, d);
            bm = om > bm ? om : bm;
            br = orr > br ? orr : br;
        }
        const float fm = __uint_as_float(bm), fr = __uint_as_float(br);
        const bool fine_m = bm < 0x7F800000u, fine_r = br < 0x7F800000u;
        const bool some_m = fine_m && fm > 7.8886090522101181e-31f, some_r = fine_r && fr > 0.0f;      // 2^-100: 127^2 / max stays finite
        const float im = some_m ? 16129.0f / fm : 0.0f, ir = some_r ? 65025.0f / fr : 0.0f;
        const unsigned kb = aw_mix((a.key[s] + (unsigned)step * AW_GOLD) ^ aw_mix((unsigned)b));
        for (int j = 0; j < 4; ++j) {
            const int e = j * 64 + lane;
            const long long i = b * AW_BLOCK + e;
            if (i >= n) continue;
            unsigned u = kb + (unsigned)e * AW_GOLD;
            u = (u ^ (u >> 16)) * 0x7FEB352Du;
            u ^= u >> 15;
            float cm = 0.0f, cr = 0.0f;
            if (some_m) cm = fminf(aw_code(fabsf(mm[j]) * im, (float)(u & 0xFFFFu) * (1.0f / 65536.0f)), 127.0f);
            if (some_r) cr = fminf(aw_code(rr[j] * ir, (float)(u >> 16) * (1.0f / 65536.0f)), 255.0f);
            if (some_r && cr == 0.0f && rr[j] > 0.0f) cr = 1.0f;
            mc[i] = (signed char)(mm[j] < 0.0f ? -(int)cm : (int)cm);
            rc[i] = (unsigned char)(int)cr;
        }
        if (lane == 0) {
            const float nan = __uint_as_float(0x7FC00000u);
            a.scales[s][2 * b] = fine_m ? (some_m ? fm / 16129.0f : 0.0f) : nan;
            a.scales[s][2 * b + 1] = fine_r ? (some_r ? fr / 65025.0f : 0.0f) : nan;
        }
    }
}

// what 8-bit moments stand for, in 32 bits: exp_avg and exp_avg_sq
__global__ __launch_bounds__(AW_THREADS) void adamw_moments_kernel(const signed char* mc, const unsigned char* rc, const float* scales,
                                                                   long long n, float* m, float* v) {
    const long long i = (long long)blockIdx.x * AW_THREADS + threadIdx.x;
    if (i >= n) return;
    const float sm = scales[2 * (i / AW_BLOCK)], sr = scales[2 * (i / AW_BLOCK) + 1];
    const float c = (float)mc[i], d = (float)rc[i], r = d * d * sr;
    m[i] = c * fabsf(c) * sm;
    v[i] = r * r;
}

template <class Args, template <int, int> class Launch>
static int aw_by_type(const Args& a, int pt, int gt, unsigned blocks, hipStream_t st) {
    if (pt == MNE_T_F32 && gt == MNE_T_F32) Launch<MNE_T_F32, MNE_T_F32>::go(a, blocks, st);
    else if (pt == MNE_T_F32 && gt == MNE_T_BF16) Launch<MNE_T_F32, MNE_T_BF16>::go(a, blocks, st);
    else if (pt == MNE_T_F32 && gt == MNE_T_F16) Launch<MNE_T_F32, MNE_T_F16>::go(a, blocks, st);
    else if (pt == MNE_T_BF16 && gt == MNE_T_F32) Launch<MNE_T_BF16, MNE_T_F32>::go(a, blocks, st);
    else if (pt == MNE_T_BF16 && gt == MNE_T_BF16) Launch<MNE_T_BF16, MNE_T_BF16>::go(a, blocks, st);
    else if (pt == MNE_T_F16 && gt == MNE_T_F32) Launch<MNE_T_F16, MNE_T_F32>::go(a, blocks, st);
    else if (pt == MNE_T_F16 && gt == MNE_T_F16) Launch<MNE_T_F16, MNE_T_F16>::go(a, blocks, st);
    else return -1;
    return 0;
}
template <int PT, int GT> struct Launch32 {
    static void go(const Adamw32Args& a, unsigned blocks, hipStream_t st) { MNE_LAUNCH((adamw32_kernel<PT, GT>), blocks, AW_THREADS, 0, st, a); }
};
template <int PT, int GT> struct Launch8 {
    static void go(const Adamw8Args& a, unsigned blocks, hipStream_t st) { MNE_LAUNCH((adamw8_kernel<PT, GT>), blocks, AW_THREADS, 0, st, a); }
};

int mne_launch_adamw32(const Adamw32Args& a, int p_type, int g_type, unsigned blocks, hipStream_t st) {
    return aw_by_type<Adamw32Args, Launch32>(a, p_type, g_type, blocks, st);
}
int mne_launch_adamw8(const Adamw8Args& a, int p_type, int g_type, unsigned blocks, hipStream_t st) {
    return aw_by_type<Adamw8Args, Launch8>(a, p_type, g_type, blocks, st);
}
int mne_launch_adamw_moments(const signed char* mc, const unsigned char* rc, const float* scales, long long n, float* m, float* v, hipStream_t st) {
    MNE_LAUNCH(adamw_moments_kernel, (unsigned)((n + AW_THREADS - 1) / AW_THREADS), AW_THREADS, 0, st, mc, rc, scales, n, m, v);
    return 0;
}
long long mne_adamw_blocks_for(long long n) { return (n + AW_PER_WG - 1) / AW_PER_WG; }
unsigned mne_adamw_key(unsigned seed, unsigned ordinal) {
    unsigned h = seed + ordinal * AW_GOLD;
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
