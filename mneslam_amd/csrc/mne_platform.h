// mne_platform.h -- the one place that decides between the real HIP toolchain (the product:
// hipcc --offload-arch=gfx950) and the test-only host emulator (tests/hostemu/hip_emu.h, used by
// the CPU test-suite to run these same kernel sources without a GPU).
#pragma once
#ifdef MNE_HOST_EMU
#include "hip_emu.h"
static inline float mne_sqrt_fast(float x) { return std::sqrt(x); }
static inline float mne_sqrt_rn(float x) { return std::sqrt(x); }
static inline float mne_rcp_fast(float x) { return 1.0f / x; }
static inline unsigned mne_max16(unsigned v) {                    // largest value of the 16 lanes of a row
    for (int d = 1; d < 16; d <<= 1) { const unsigned o = __shfl_xor(v, d); v = o > v ? o : v; }
    return v;
}
static inline float mne_quad(float v, int k) { return __shfl(v, (int)(threadIdx.x & 60u) | k); }      // lane k's of every four lanes
static inline unsigned mne_pack4(unsigned a, unsigned b, unsigned c, unsigned d) { return (a & 255u) | (b & 255u) << 8 | (c & 255u) << 16 | d << 24; }
static inline int mne_first_lane(int v) { return __shfl(v, 0); }
// bf16 <-> fp32, rounded to nearest even
static inline float mne_bf16_to_float(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
static inline unsigned short mne_float_to_bf16(float x) {
    const unsigned u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (unsigned short)((u >> 16) | 0x40u);
    return (unsigned short)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
#else
#include <hip/hip_runtime.h>
#define MNE_LAUNCH(kern, grid, block, lds, stream, ...) \
    hipLaunchKernelGGL(kern, dim3(grid), dim3(block), lds, stream, __VA_ARGS__)
#define hipLaunchOrEmu2D(kern, gx, gy, block, stream, ...) hipLaunchKernelGGL(kern, dim3(gx, gy), dim3(block), 0, stream, __VA_ARGS__)
#define MNE_LDS_MAX (160 * 1024)      // LDS per CU on gfx950
// inter-workgroup hand-off inside one launch (cdna_hip_programming.md, Guideline 16): drain this wave's stores, agent-scope
// release / acquire by one lane
#define MNE_DRAIN_STORES() asm volatile("s_waitcnt vmcnt(0)" ::: "memory")
#define MNE_FENCE_RELEASE_AGENT() __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent")
#define MNE_FENCE_ACQUIRE_AGENT() __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent")
#define MNE_SET_MAX_LDS(kern, bytes) (void)hipFuncSetAttribute((const void*)(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)(bytes))
#define MNE_DYN_LDS(name) extern __shared__ __attribute__((aligned(16))) unsigned char name[]
// Decoder weights are wave-uniform: reading them through the constant address space makes the
// compiler use scalar (SMEM) loads, so the tiny-MLP FMAs take their weight operand from SGPRs.
typedef const __attribute__((address_space(4))) float* mne_cptr;
#define MNE_CPTR(p) ((mne_cptr)(unsigned long long)(p))
// Broadcast of lane k (0..7, compile-time) inside every aligned group of 8 lanes: ds_swizzle in bit-mask mode,
// new_lane = (lane & 0x18) | k within each half-wave; goes through the LDS crossbar, touches no LDS memory.
#define MNE_SWZ8(k) (0x18 | ((k) << 5))
static __device__ __forceinline__ int mne_bcast8(int v, int k) {
    switch (k) {      // the pattern must be an immediate
        case 0: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(0));
        case 1: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(1));
        case 2: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(2));
        case 3: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(3));
        case 4: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(4));
        case 5: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(5));
        case 6: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(6));
        default: return __builtin_amdgcn_ds_swizzle(v, MNE_SWZ8(7));
    }
}
static __device__ __forceinline__ float mne_bcast8(float v, int k) { return __int_as_float(mne_bcast8(__float_as_int(v), k)); }
static __device__ __forceinline__ float mne_sqrt_fast(float x) { return __builtin_amdgcn_sqrtf(x); }      // v_sqrt_f32: 1 ulp
// The root rounded to nearest, for 0, 2^-96 and above, infinity and NaN: of s (1 ulp off) and its neighbours the one whose product with
// the next lower one is below x and with the next higher one is not (between neighbours s < t: x > s t puts the root above their middle).
static __device__ __forceinline__ float mne_sqrt_rn(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float lo = __int_as_float(__float_as_int(s) - 1), hi = __int_as_float(__float_as_int(s) + 1);
    float r = fmaf(-lo, s, x) <= 0.0f ? lo : s;
    return fmaf(-hi, s, x) > 0.0f ? hi : r;
}
static __device__ __forceinline__ float mne_rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }        // v_rcp_f32: 1 ulp
// largest value of the 16 lanes of a row: four rotations within the row, no LDS
template <int CTRL> static __device__ __forceinline__ unsigned mne_max_ror(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}
// lane k's value (a constant) of every four lanes
static __device__ __forceinline__ float mne_quad(float v, int k) {
    const int x = __float_as_int(v);
    switch (k) {
        case 0: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x00, 0xF, 0xF, true));
        case 1: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x55, 0xF, 0xF, true));
        case 2: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0xAA, 0xF, 0xF, true));
        default: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0xFF, 0xF, 0xF, true));
    }
}
// the lowest bytes of four words
static __device__ __forceinline__ unsigned mne_pack4(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}
static __device__ __forceinline__ int mne_first_lane(int v) { return __builtin_amdgcn_readfirstlane(v); }
static __device__ __forceinline__ unsigned mne_max16(unsigned v) {
    return mne_max_ror<0x121>(mne_max_ror<0x122>(mne_max_ror<0x124>(mne_max_ror<0x128>(v))));
}
static __device__ __forceinline__ float mne_bf16_to_float(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
static __device__ __forceinline__ unsigned short mne_float_to_bf16(float x) {         // one v_cvt_pk_bf16_f32: to nearest even
    return __builtin_bit_cast(unsigned short, (__bf16)x);
}
// The XCD (accelerator complex die, 0..7 on MI355X) this wave runs on: hardware register XCC_ID.
static __device__ __forceinline__ int mne_xcc_id() {
    int v;
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(v));
    return v & 7;
}
// LDS hand-off between the lanes of ONE wave (each wave owns a private LDS region): DS operations of
// a wave complete in issue order, so draining lgkmcnt and pinning the compiler's order is enough --
// no s_barrier, the four waves of a workgroup never wait for each other.
// pin the instruction scheduler at this point (nothing moves across it)
#define MNE_SCHED_BARRIER() __builtin_amdgcn_sched_barrier(0)
#define MNE_WAVE_SYNC()                                         \
    do {                                                        \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      \
        __builtin_amdgcn_wave_barrier();                        \
    } while (0)
#endif

// B bytes of memory, at any address, that are loaded and stored as one (global memory takes them so whatever their alignment)
template <int B> struct MneBytes;
template <> struct MneBytes<16> { typedef unsigned words __attribute__((ext_vector_type(4), aligned(1))); words v; };
template <> struct MneBytes<8> { typedef unsigned words __attribute__((ext_vector_type(2), aligned(1))); words v; };
template <> struct MneBytes<4> { typedef unsigned words __attribute__((aligned(1))); words v; };
// of data that nothing reads again soon: it leaves the caches to others
template <int B> static __device__ __forceinline__ MneBytes<B> mne_load_once(const MneBytes<B>* p) {
    MneBytes<B> x;
    x.v = __builtin_nontemporal_load(&p->v);
    return x;
}
template <int B> static __device__ __forceinline__ void mne_store_once(MneBytes<B>* p, const MneBytes<B>& x) { __builtin_nontemporal_store(x.v, &p->v); }

// the unsigned integer of B bytes
template <int B> struct MneWord;
template <> struct MneWord<4> { typedef unsigned type; };
template <> struct MneWord<2> { typedef unsigned short type; };
