// Device helpers of the sequence operators (layer_norm.hip, causal_conv.hip, scan.hip): rows of float, bf16 or f16
// elements are moved V at a time, up to 16 bytes, the arithmetic is f32, and each result is rounded once, to nearest even,
// when it is stored.
#pragma once
#include "common.h"

template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float x) { return (_Float16)x; }

template <typename T, int V> struct RowVec { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T> struct RowVec<T, 1> { typedef T type; };

// V consecutive elements as they lie in memory, at any element's address (one access: the hardware takes vector loads and
// stores of global memory at any alignment, so an odd width does not cost the wide accesses)
template <typename T, int V> struct Raw {
    typename RowVec<T, V>::type v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const typename RowVec<T, V>::type*>(p); }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (V == 1) return to_f32(v); else return to_f32((T)v[i]);
    }
    __device__ __forceinline__ void zero() {
        if constexpr (V == 1) v = from_f32<T>(0.f);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void set(int i, float x) {
        if constexpr (V == 1) v = from_f32<T>(x); else v[i] = from_f32<T>(x);
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename RowVec<T, V>::type*>(p) = v; }
};

// Buffer accesses: a uniform base in scalar registers and a 32-bit byte offset per lane; an offset of BUF_OUT reads zeros
// and writes nothing (the range check of the hardware), which is how rows and channels past the end are left out.
constexpr unsigned BUF_OUT = 0x80000000u, BUF_BYTES = 0x7fffffffu;
template <typename T, int V> __device__ __forceinline__ Raw<T, V> buf_load(__amdgpu_buffer_rsrc_t r, unsigned off) {
    constexpr int N = V * sizeof(T);
    Raw<T, V> o;
    if constexpr (N == 16) o.v = __builtin_bit_cast(typename RowVec<T, V>::type, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    else if constexpr (N == 8) o.v = __builtin_bit_cast(typename RowVec<T, V>::type, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    else if constexpr (N == 4) o.v = __builtin_bit_cast(typename RowVec<T, V>::type, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    else o.v = __builtin_bit_cast(typename RowVec<T, V>::type, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
    return o;
}
template <typename T, int V> __device__ __forceinline__ void buf_store(__amdgpu_buffer_rsrc_t r, unsigned off, const Raw<T, V>& o) {
    constexpr int N = V * sizeof(T);
    if constexpr (N == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o.v), r, off, 0, 0);
    else if constexpr (N == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, o.v), r, off, 0, 0);
    else if constexpr (N == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, o.v), r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, o.v), r, off, 0, 0);
}

// exp through the hardware's base-2 exponential (1 ulp; results under 2^-126 become 0)
__device__ __forceinline__ float exp_f(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.f + exp_f(-x)); }
// x * sigmoid(x): exp(-x) may overflow to infinity, whose reciprocal is the 0 that is meant
__device__ __forceinline__ float silu_f(float x) { return x * sigmoid_f(x); }
__device__ __forceinline__ float dsilu_f(float x) {
    const float s = sigmoid_f(x);
    return s * (1.f + x * (1.f - s));
}

static inline int vqa_elem_bytes(int dtype) { return dtype == VQA_F32 ? 4 : 2; }
static inline bool vqa_dtype_ok(int dtype) { return dtype == VQA_F32 || dtype == VQA_BF16 || dtype == VQA_F16; }
// a pointer whose rows start `stride` elements apart can be read `bytes` at a time
static inline bool vqa_vec_ok(const void* p, long stride, int elem, int bytes = 16) {
    return ((uintptr_t)p & (bytes - 1)) == 0 && (stride * elem) % bytes == 0;
}

// Column sums of part[rows][cols] (f32) in a fixed order: 32 columns x 32 row lanes per workgroup, eight rows of each lane
// in flight, the lanes joined through LDS.  Column c of the first `n0` goes to out0[c], the rest to out1[c - n0].
__global__ __launch_bounds__(1024) static void seq_column_sums(const float* __restrict__ part, int rows, long cols,
                                                               float* __restrict__ out0, long n0,
                                                               float* __restrict__ out1) {
    const int lc = threadIdx.x & 31, lane_row = threadIdx.x >> 5;
    const long c = (long)blockIdx.x * 32 + lc;
    float acc[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u] = 0.f;
    if (c < cols) {
        for (int r = lane_row; r < rows; r += 256) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (r + 32 * u < rows) acc[u] += part[(long)(r + 32 * u) * cols + c];
        }
    }
    __shared__ float s[32][33];
    s[lane_row][lc] = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
    __syncthreads();
    if (lane_row == 0 && c < cols) {
        float t = 0.f;
#pragma unroll
        for (int u = 0; u < 32; ++u) t += s[u][lc];
        if (c < n0) { if (out0) out0[c] = t; }
        else if (out1) out1[c - n0] = t;
    }
}
static inline void seq_sum_columns(hipStream_t st, const float* part, int rows, long cols, float* out0, long n0,
                                   float* out1) {
    seq_column_sums<<<(unsigned)((cols + 31) / 32), 1024, 0, st>>>(part, rows, cols, out0, n0, out1);
}
