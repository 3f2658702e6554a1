// What the kernels of it_tree_attention share (it_tree_attention.cu: host side, mma.sync kernels; it_tree_attention_tc.cu: tcgen05 kernels).
#pragma once
#include "it_ops.cuh"
#include "it_pipe.cuh"
#include <type_traits>

// What a kernel of a call gets.
struct TaParams {
    const void *q, *gate; void* out; const int *parents, *length; float* weights;
    float* part_o; float2* part_ml; float2* stats; int* status;
    long long q_row, q_head, g_row, g_head, o_row, o_head, w_head;
    int rows, heads, group, kv_heads, dim, cached, splits, prows, pad_rows; float scale;
};

// it_tree_attention_tc.cu.  nb: 64-element pieces of a head, nr: product rows of a CTA (16, 32 or 64).
int it_tree_tc_prepare();
int it_tree_tc_run(const TaParams& p, int type, int nb, int nr, int row_tiles, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st);
int it_tree_tc_weigh(const TaParams& p, int type, int nb, int nr, const CUtensorMap& km, cudaStream_t st);

namespace {

constexpr int TA_KEYS = 64, TA_MAXROWS = 256, TA_WORDS = TA_MAXROWS / 32, TA_UNIT_MAX = 8;
constexpr int TA_SMEM_MAX = 226 * 1024;
constexpr float TA_LOG2E = 1.4426950408889634f;
constexpr float TA_SHIFT = 14.f;         // p is 2^14 at the maximum: small ones keep their bits in f16

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <class T> struct Ta16;
template <> struct Ta16<__half> {
    static constexpr unsigned EXP = 0x7c00u;
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const unsigned*>(&h); }
    static __device__ __forceinline__ float2 unpack(unsigned u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Ta16<__nv_bfloat16> {
    static constexpr unsigned EXP = 0x7f80u;
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const unsigned*>(&h); }
    static __device__ __forceinline__ float2 unpack(unsigned u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
// The two values of a register with non-finite ones replaced by zero; `seen` collects whether there were any.
template <class T> __device__ __forceinline__ unsigned finite_only(unsigned u, bool& seen) {
    const bool lo = (u & Ta16<T>::EXP) == Ta16<T>::EXP, hi = ((u >> 16) & Ta16<T>::EXP) == Ta16<T>::EXP;
    seen = seen || lo || hi;
    return u & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
}
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], unsigned a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void tma_load_3d(unsigned dst, const void* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// Place of 16-byte piece c (0..7) of row r in a box of 128-byte rows with the 128-byte swizzle.
__device__ __forceinline__ unsigned swz(int r, int c) { return (unsigned)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Cached slots of this call, and all its slots.
__device__ __forceinline__ int ta_cached(const TaParams& p) { return p.length ? min(max(*p.length, 0), p.cached) : p.cached; }

// Which rows each row sees, as bits: its parent's set and itself, by following pointers twice as far in every round.  Ends after the rounds it takes
// for `rows` rows whatever the pointers are; a parent that is not a smaller row counts as none.
__device__ void ta_ancestors(unsigned (*anc)[TA_WORDS], int* jump, const int* parents, int rows) {
    const int tid = threadIdx.x, n = blockDim.x;
    for (int t = tid; t < rows; t += n) {
        const int q = parents[t];
        jump[t] = q >= 0 && q < t ? q : -1;
#pragma unroll
        for (int w = 0; w < TA_WORDS; w++) anc[t][w] = w == t >> 5 ? 1u << (t & 31) : 0u;
    }
    __syncthreads();
    for (int far = 1; far < rows; far <<= 1) {
        unsigned add[2][TA_WORDS]; int next[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {                       // at least 128 threads: two rows each at most
            const int t = tid + k * n, j = t < rows ? jump[t] : -1;
            next[k] = j >= 0 ? jump[j] : -1;
#pragma unroll
            for (int w = 0; w < TA_WORDS; w++) add[k][w] = j >= 0 ? anc[j][w] : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int t = tid + k * n;
            if (t >= rows) continue;
            jump[t] = next[k];
#pragma unroll
            for (int w = 0; w < TA_WORDS; w++) anc[t][w] |= add[k][w];
        }
        __syncthreads();
    }
}


// Eight elements of a product row per lane: high and, for f32 activations, low halves, and the factor from products with them to log2 of the exponential.
template <class T, bool SPLIT>
__device__ __forceinline__ float ta_q_row(const TaParams& p, bool live, int t, int h, int lane, unsigned (&hi)[4], unsigned (&lo)[4]) {
    float f = p.scale * TA_LOG2E;
    if constexpr (SPLIT) {
        float v[8] = {};
        if (live) {
            const float* x = (const float*)p.q + t * p.q_row + h * p.q_head + 8 * lane;
            float a[4], b[4]; load4(x, a); load4(x + 4, b);
#pragma unroll
            for (int j = 0; j < 4; j++) { v[j] = a[j]; v[4 + j] = b[j]; }
        }
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[j]));
#pragma unroll
        for (int s = 16; s; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        // 2^e brings the row's largest element to [2^14, 2^15): the low halves keep 22 bits of it without leaving f16's range
        const int e = min(max(14 - ((int)(__float_as_uint(m) >> 23) - 127), -110), 110);
        const float up = __uint_as_float((unsigned)(127 + e) << 23);
        f *= __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float a = v[2 * j] * up, b = v[2 * j + 1] * up;
            hi[j] = Ta16<T>::pack(a, b);
            const float2 h2 = Ta16<T>::unpack(hi[j]);
            lo[j] = Ta16<T>::pack(a - h2.x, b - h2.y);
        }
    } else if (live) {
        const uint2* x = reinterpret_cast<const uint2*>((const T*)p.q + t * p.q_row + h * p.q_head + 8 * lane);
        const uint2 a = x[0], b = x[1];
        hi[0] = a.x; hi[1] = a.y; hi[2] = b.x; hi[3] = b.y;
    }
    return f;
}

// A launch that may begin while the kernel before it in the stream still runs; it waits for that kernel itself.
template <typename... KArgs, typename... Args> cudaError_t ta_launch(bool early, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Whether row t sees slot j.
__device__ __forceinline__ bool ta_sees(const TaParams& p, const unsigned (*anc)[TA_WORDS], int t, int j, int cached) {
    const int i = j - cached;
    if (i < 0) return true;
    if (i >= p.rows) return false;
    return p.parents ? (anc[t][i >> 5] >> (i & 31)) & 1u : i <= t;
}

}  // namespace
