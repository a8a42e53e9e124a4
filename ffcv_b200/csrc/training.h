// What the kernels of the training step share (cross_entropy.cu, norm_residual.cu, rotary.cu, adamw.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/ffcv_b200.h"

namespace ffcvb {

constexpr int kSms = 148;

// The message of the calling thread's last failure; returns `code`.
int training_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

// Makes `device` current for a call's launches, and the one before it again afterwards.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
        ok_ = before_ == device || cudaSetDevice(device) == cudaSuccess;
        if (before_ == device) before_ = -1;
    }
    ~OnDevice() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    bool ok() const { return ok_; }

  private:
    int before_ = -1;
    bool ok_ = false;
};

inline int launched(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FFCVB_OK : training_fail(FFCVB_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Calls f with a value of the type that a FFCVB_TYPE_* stands for.
template <typename F>
bool with_type(int type, F &&f) {
    switch (type) {
    case FFCVB_TYPE_F32: f(float{}); return true;
    case FFCVB_TYPE_F16: f(__half{}); return true;
    case FFCVB_TYPE_BF16: f(__nv_bfloat16{}); return true;
    }
    return false;
}
inline int type_size(int type) { return type == FFCVB_TYPE_F32 ? 4 : 2; }

#ifdef __CUDACC__

// Programmatic launches, of all kernels here: such a kernel may begin once every CTA of the one before it has called let_next_begin() or
// ended; it calls wait_for_previous() before it touches what earlier kernels of the stream wrote or read.  What it saves is the way from one
// kernel's end to the next one's begin (rotary, queries and keys forward and backward in turn, 65 us each: 141 us a pair without, 137 with).
template <typename... Params, typename... Given>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t room, cudaStream_t stream, Given &&...given) {
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    how.gridDim = grid;
    how.blockDim = block;
    how.dynamicSmemBytes = room;
    how.stream = stream;
    how.attrs = &early;
    how.numAttrs = 1;
    return cudaLaunchKernelEx(&how, kernel, static_cast<Params>(given)...);
}
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N values that are loaded and stored at once: 16 bytes of them, or one.
template <typename T, int N> struct Pack;
template <typename T> struct Pack<T, 1> {
    T raw;
    __device__ __forceinline__ void load(const T *p) { raw = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = raw; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_float(raw); }
    __device__ __forceinline__ void set(const float (&v)[1]) { raw = from_float<T>(v[0]); }
};
template <typename T> struct Pack16 {
    uint4 raw;
    __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = raw; }
};
// Half as much: 8 bytes.
template <typename T> struct Pack8 {
    uint2 raw;
    __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint2 *>(p) = raw; }
};
template <> struct Pack<float, 2> : Pack8<float> {
    __device__ __forceinline__ void get(float (&v)[2]) const {
        v[0] = __uint_as_float(raw.x);
        v[1] = __uint_as_float(raw.y);
    }
    __device__ __forceinline__ void set(const float (&v)[2]) { raw = make_uint2(__float_as_uint(v[0]), __float_as_uint(v[1])); }
};
template <> struct Pack<__nv_bfloat16, 4> : Pack8<__nv_bfloat16> {
    __device__ __forceinline__ void get(float (&v)[4]) const {
        v[0] = __uint_as_float(raw.x << 16);
        v[1] = __uint_as_float(raw.x & 0xffff0000u);
        v[2] = __uint_as_float(raw.y << 16);
        v[3] = __uint_as_float(raw.y & 0xffff0000u);
    }
    __device__ __forceinline__ void set(const float (&v)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        raw = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};
template <> struct Pack<__half, 4> : Pack8<__half> {
    __device__ __forceinline__ void get(float (&v)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
    __device__ __forceinline__ void set(const float (&v)[4]) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        raw = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};
template <> struct Pack<float, 4> : Pack16<float> {
    __device__ __forceinline__ void get(float (&v)[4]) const {
        v[0] = __uint_as_float(raw.x);
        v[1] = __uint_as_float(raw.y);
        v[2] = __uint_as_float(raw.z);
        v[3] = __uint_as_float(raw.w);
    }
    __device__ __forceinline__ void set(const float (&v)[4]) {
        raw = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Pack<__nv_bfloat16, 8> : Pack16<__nv_bfloat16> {
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[2 * k] = __uint_as_float(w[k] << 16);
            v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&two);
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Pack<__half, 8> : Pack16<__half> {
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            v[2 * k] = two.x;
            v[2 * k + 1] = two.y;
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __half2 two = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&two);
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

#endif

} // namespace ffcvb
