// What the kernels of it_tree_attention share (it_tree_attention.cu: host side and the joining of runs; it_tree_attention_tc.cu: the products).
#pragma once
#include "it_ops.cuh"
#include "it_pipe.cuh"
#include <type_traits>

// What a kernel of a call gets.
struct TaParams {
    const void *q, *gate; void* out; const int *parents, *length; float* weights;
    float* part_o; float2* part_ml; float2* stats; float* scores; int* status;          // scores: [kv head][product row][slot] in log2 units, null if they are not kept
    long long q_row, q_head, g_row, g_head, o_row, o_head, w_head, s_row;
    int rows, heads, group, kv_heads, dim, cached, splits, prows, pad_rows, joined, tile_warps; unsigned group_inv; float scale;
};

// it_tree_attention_tc.cu.  nb: 64-element pieces of a head, nr: product rows of a CTA (16, 32 or 64).
int it_tree_tc_prepare();
int it_tree_tc_run(const TaParams& p, int type, int nb, int nr, int row_tiles, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st);
int it_tree_tc_weigh(const TaParams& p, int type, int nb, const CUtensorMap& km, cudaStream_t st);

namespace {

constexpr int TA_KEYS = 128, TA_MAXROWS = 256, TA_WORDS = TA_MAXROWS / 32, TA_MAXSPLITS = 148;       // slots of a tile; rows of a call; runs of a cache, one an SM
constexpr float TA_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <class T> struct Ta16;
template <> struct Ta16<__half> {
    static constexpr unsigned EXP = 0x7c00u;
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const unsigned*>(&h); }
    static __device__ __forceinline__ float2 unpack(unsigned u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
};
template <> struct Ta16<__nv_bfloat16> {
    static constexpr unsigned EXP = 0x7f80u;
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const unsigned*>(&h); }
    static __device__ __forceinline__ float2 unpack(unsigned u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
};
__device__ __forceinline__ void tma_load_3d(unsigned dst, const void* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// Place of 16-byte piece c (0..7) of row r in a box of 128-byte rows with the 128-byte swizzle.
__device__ __forceinline__ unsigned swz(int r, int c) { return (unsigned)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Cached slots of this call, and all its slots.
__device__ __forceinline__ int ta_cached(const TaParams& p) { return p.length ? min(max(*p.length, 0), p.cached) : p.cached; }

// Which rows each row sees, as bits: its parent's set and itself, by following pointers twice as far in every round.  N threads, `sync` a barrier of theirs.  Ends after
// the rounds it takes for `rows` rows whatever the pointers are; a parent that is not a smaller row counts as none.
template <int N, class F>
__device__ __forceinline__ void ta_ancestors(unsigned (*anc)[TA_WORDS], int* jump, const int* parents, int rows, int tid, F sync) {
    static_assert(N >= TA_MAXROWS, "a row a thread");
    const bool live = tid < rows;
    if (live) {
        const int q = parents[tid];
        jump[tid] = q >= 0 && q < tid ? q : -1;
#pragma unroll
        for (int w = 0; w < TA_WORDS; w++) anc[tid][w] = w == tid >> 5 ? 1u << (tid & 31) : 0u;
    }
    sync();
    const int words = (rows + 31) / 32;
#pragma unroll 1
    for (int far = 1; far < rows; far <<= 1) {
        unsigned add[TA_WORDS];
        const int j = live ? jump[tid] : -1, next = j >= 0 ? jump[j] : -1;
#pragma unroll
        for (int w = 0; w < TA_WORDS; w++) add[w] = j >= 0 && w < words ? anc[j][w] : 0u;
        sync();
        if (live) {
            jump[tid] = next;
#pragma unroll
            for (int w = 0; w < TA_WORDS; w++) if (w < words) anc[tid][w] |= add[w];
        }
        sync();
    }
}

// Row t of product row r: r / group, by a product (exact: r < 2^18, group <= 2^10).
__device__ __forceinline__ int ta_row(const TaParams& p, int r) { return p.group == 1 ? r : (int)__umulhi((unsigned)r, p.group_inv); }

// Eight elements of a product row per lane; halves(): as f16 or bf16, for f32 activations the high and low halves, and the factor from products with them to log2 of the
// exponential.
template <class T, bool SPLIT> struct TaRow;
template <class T> struct TaRow<T, false> {
    uint2 a, b;
    __device__ __forceinline__ void load(const TaParams& p, bool live, int t, int h, int lane) {
        a = b = make_uint2(0u, 0u);
        if (live) { const uint2* x = reinterpret_cast<const uint2*>((const T*)p.q + t * p.q_row + h * p.q_head + 8 * lane); a = x[0]; b = x[1]; }
    }
    __device__ __forceinline__ float halves(const TaParams& p, unsigned (&hi)[4], unsigned (&)[4]) const { hi[0] = a.x; hi[1] = a.y; hi[2] = b.x; hi[3] = b.y; return p.scale * TA_LOG2E; }
};
template <class T> struct TaRow<T, true> {
    float4 a, b;
    __device__ __forceinline__ void load(const TaParams& p, bool live, int t, int h, int lane) {
        a = b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live) { const float4* x = reinterpret_cast<const float4*>((const float*)p.q + t * p.q_row + h * p.q_head + 8 * lane); a = x[0]; b = x[1]; }
    }
    __device__ __forceinline__ float halves(const TaParams& p, unsigned (&hi)[4], unsigned (&lo)[4]) const {
        const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[j]));
        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));       // not negative: the bits are in the floats' order
        // 2^e brings the row's largest element to [2^14, 2^15): the low halves keep 22 bits of it without leaving f16's range
        const int e = min(max(14 - ((int)(__float_as_uint(m) >> 23) - 127), -110), 110);
        const float up = __uint_as_float((unsigned)(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = v[2 * j] * up, y = v[2 * j + 1] * up;
            hi[j] = Ta16<T>::pack(x, y);
            const float2 h2 = Ta16<T>::unpack(hi[j]);
            lo[j] = Ta16<T>::pack(x - h2.x, y - h2.y);
        }
        return p.scale * TA_LOG2E * __uint_as_float((unsigned)(127 - e) << 23);
    }
};

// Whether row t sees slot j.
__device__ __forceinline__ bool ta_sees(const TaParams& p, const unsigned (*anc)[TA_WORDS], int t, int j, int cached) {
    const int i = j - cached;
    if (i < 0) return true;
    if (i >= p.rows) return false;
    return p.parents ? (anc[t][i >> 5] >> (i & 31)) & 1u : i <= t;
}

}  // namespace
