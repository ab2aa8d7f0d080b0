// Element types of the token-model operators: 16-byte vectors of fp32 / fp16 / bf16 as floats, rows whose start
// is no multiple of 16 bytes, warp and block sums.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nzb {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <>
struct Elem<__half> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// A row of n elements seen as 16-byte blocks of memory: block v holds the elements v * VEC - lead ..
// v * VEC - lead + VEC - 1, where `lead` is how many elements before the row share its first block. Blocks
// that lie whole within the row are moved as one vector, the first and the last one element by element, so
// nothing outside the row is touched.
template <typename T>
__device__ __forceinline__ int row_lead(const T* row) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
template <typename T>
__device__ __forceinline__ uint4 load_block(const T* row, int64_t first, int64_t n) {
    constexpr int VEC = Elem<T>::VEC;
    if (first >= 0 && first + VEC <= n) return *reinterpret_cast<const uint4*>(row + first);
    union { uint4 u; T e[VEC]; } b;
    b.u = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < VEC; i++)
        if (first + i >= 0 && first + i < n) b.e[i] = row[first + i];
    return b.u;
}
template <typename T>
__device__ __forceinline__ void store_block(T* row, int64_t first, int64_t n, const uint4& v) {
    constexpr int VEC = Elem<T>::VEC;
    if (first >= 0 && first + VEC <= n) {
        *reinterpret_cast<uint4*>(row + first) = v;
        return;
    }
    union { uint4 u; T e[VEC]; } b;
    b.u = v;
#pragma unroll
    for (int i = 0; i < VEC; i++)
        if (first + i >= 0 && first + i < n) row[first + i] = b.e[i];
}

// Two fp32 operations in one instruction (sm_100): the elementwise work of 16-bit rows is bound by issue slots.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Programmatic launch: a kernel may start while the one before it on the stream ends, and waits here until that one has
// ended and its writes are visible.
__device__ __forceinline__ void kernel_wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void kernel_allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Launches such a kernel.
template <typename... Params, typename... Args>
inline cudaError_t launch_programmatic(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Runs the statement with T as the element type that `dtype` names.
#define NZB_DISPATCH_DTYPE(dtype, T, ...)                                             \
    do {                                                                              \
        if ((dtype) == NZB_F32) { using T = float; __VA_ARGS__; }                     \
        else if ((dtype) == NZB_F16) { using T = __half; __VA_ARGS__; }               \
        else { using T = __nv_bfloat16; __VA_ARGS__; }                                \
    } while (0)

inline bool known_dtype(int32_t t) { return t == 0 || t == 1 || t == 2; }
inline int64_t dtype_size(int32_t t) { return t == 0 ? 4 : 2; }
inline int64_t index_size(int32_t t) { return t == 0 ? 4 : 8; }
inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace nzb
