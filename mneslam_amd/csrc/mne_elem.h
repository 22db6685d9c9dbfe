// mne_elem.h -- elements in memory (fp32, bf16, fp16; MNE_T_*) as the fp32 numbers that kernels compute with.
#pragma once
#include "mne_platform.h"
#include "mneslam_hip.h"

template <int T> struct MneElem;
template <> struct MneElem<MNE_T_F32> {
    typedef float mem;
    static __device__ __forceinline__ float get(mem x) { return x; }
    static __device__ __forceinline__ mem put(float x) { return x; }
};
template <> struct MneElem<MNE_T_BF16> {
    typedef unsigned short mem;
    static __device__ __forceinline__ float get(mem x) { return mne_bf16_to_float(x); }
    static __device__ __forceinline__ mem put(float x) { return mne_float_to_bf16(x); }
};
template <> struct MneElem<MNE_T_F16> {
    typedef _Float16 mem;
    static __device__ __forceinline__ float get(mem x) { return (float)x; }
    static __device__ __forceinline__ mem put(float x) { return (_Float16)x; }
};
