// What the operators of the attention block (it_norm_rope.cu, it_tree_attention.cu, it_cache_evict.cu) share: they take raw device pointers
// and a stream instead of a context, so the device's facts and the word in which a kernel says that a wait ran out live here.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "it_internal.h"

// The current device's SM count and status word (mapped host memory, made by the first call on the device: not while `stream` is recorded).
struct it_ops_device { int device, sm_count; int *status_host, *status_dev; };
int it_ops_current(void* stream, const char* who, it_ops_device* out);

static inline bool it_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
static inline size_t it_type_size(int type) { return type == IT_F32 ? 4 : 2; }
// Activations over a cache: f32 over f16, or one 16-bit type for both.
static inline bool it_type_pair(int act, int cache) { return (act == IT_F32 && cache == IT_F16) || (act == IT_F16 && cache == IT_F16) || (act == IT_BF16 && cache == IT_BF16); }
// Whether [a, a + an) and [b, b + bn) share a byte.
static inline bool it_overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + bn && y < x + an;
}
// A stretch of memory that a call reads or writes, and the first of `others` (n of them) that shares a byte with it; null if none does.
struct it_stretch { const char* name; const void* at; size_t bytes; };
static inline const char* it_overlaps(const it_stretch& a, const it_stretch* others, int n) {
    for (int i = 0; i < n; i++) if (a.at && others[i].at && a.bytes && others[i].bytes && it_overlap(a.at, a.bytes, others[i].at, others[i].bytes)) return others[i].name;
    return nullptr;
}
// Bytes from the first to behind the last element of a [n0][n1][d] array with these strides.
static inline size_t it_span(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t d, size_t size) {
    return n0 > 0 && n1 > 0 ? ((size_t)(n0 - 1) * (size_t)s0 + (size_t)(n1 - 1) * (size_t)s1 + (size_t)d) * size : 0;
}
// Strides of a [n0][n1][d] array that nothing overlaps itself with: the smaller one holds a head, the larger one all of the other axis.
static inline bool it_strides_ok(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t d, int64_t unit) {
    const int64_t most = (int64_t)1 << 38;                     // below the 2^40 bytes of a tensor map's stride
    if ((n0 > 1 && (s0 < d || s0 % unit || s0 >= most)) || (n1 > 1 && (s1 < d || s1 % unit || s1 >= most))) return false;
    return n0 <= 1 || n1 <= 1 || (s0 <= s1 ? s1 >= (n0 - 1) * s0 + d : s0 >= (n1 - 1) * s1 + d);
}

// A launch that may begin while the kernel before it in the stream still runs.  The first kernel of every call waits (griddepcontrol.wait) before it touches global memory, and the later ones
// before they touch what the call writes, so that a chain of them is ordered like plain launches; what overlaps is the launch itself and the kernel's start (1.5 us of a short call).
// A kernel whose successors read the caller's tensors before their wait must not let them begin before its own.
template <typename... KArgs, typename... Args> static inline cudaError_t it_launch_early(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension; attr[1].val.clusterDim.x = (unsigned)cluster; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

namespace {
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// Four neighbouring elements as one access.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) { const float4 a = *reinterpret_cast<const float4*>(p); v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; }
template <class T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
    union { uint2 u; T e[4]; } a; a.u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f32(a.e[i]);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <class T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    union { uint2 u; T e[4]; } a;
#pragma unroll
    for (int i = 0; i < 4; i++) a.e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint2*>(p) = a.u;
}
}  // namespace
