// Attention of a token, a chain or a tree of drafted tokens over a KV cache that the caller owns: host side, and the kernels that join runs of the cache and form received weights.  Stands where
// VkEngine records its attention dispatch (src/vk/mod.rs:833-840; CPU: src/cpu.rs:177-186), for any strides and lengths; sums are those of a softmax over runs of
// the cache, not the reference's position order.
//
//   p = softmax(scale q.k) over the slots that a row sees,   out = (p v) * sigmoid(gate),   weights[g][slot] += sum of p over rows and heads of g
//
// One pass over K and V.  All rows and query heads of a KV head share its keys, so they are the columns of one matrix product ("product rows": row t * group + head).
// The cache is cut into runs of 128-slot tiles, one per CTA (k_tree_attention_tc, it_tree_attention_tc.cu), so that a single token's few product rows still use every SM, and
// k_tree_join puts the runs' sums together; a cache of one tile is finished by its CTA.
// f32 activations: q (scaled per row by a power of two to the top of f16's range) and p are each the sum of two f16 values, 22 bits, and every product is
// done twice; the f16 cache is exact.  16-bit activations: q is exact, p is two values of the cache's type (22 bits, bf16 16), so that a result is rounded once, when it is stored.
// Masks: only tiles that reach behind the cached slots look at them.  A masked score is replaced, whatever it was; there a non-finite V element is
// taken out of the product and added to the rows that do see it (0 * inf would be NaN in those that do not).
// Received weights need the finished references and sums: the one pass leaves its scores, and a small kernel turns them into weights; where the scores would take too much
// memory, K is walked a second time (k_tree_weights_tc).
#include "it_tree_attention.cuh"
#include "it_route.h"
#include <mutex>

namespace {

constexpr int TA_JOINROWS = 8;                    // product rows whose received weights are formed beside the joining of runs, at most

// weights[g][slot] += ex2(score - reference) / sum over the product rows, from the scores that k_tree_attention_tc left.  CTA b has one tile of slots or, where the rows are few, several; a lane
// has four slots, and the sums of the warps that share a tile meet in a fixed order.  Latency and L2: 4 bytes a row and slot, written and read, in place of a second walk over K with its
// products (9 rows at 8192 slots: 30.5 us for the call with the walk).  JOIN: references and sums are those of runs, and joined here, so that few rows' weights need not wait for a kernel more;
// many rows' would be read by every CTA (60 rows at 30,000 slots: 68 us for the call against 49).
template <int WARPS, bool JOIN> __device__ __forceinline__ void ta_weigh(const TaParams& p, int b, int g, int tid) {
    __shared__ float part[WARPS][TA_KEYS];
    __shared__ float2 stat[JOIN ? TA_JOINROWS : 1];
    const int warp = tid >> 5, lane = tid & 31, groups = p.tile_warps, first = warp % groups, tile = b * (WARPS / groups) + warp / groups;
    const int total = ta_cached(p) + p.rows, rows = tile * TA_KEYS < total ? p.prows : 0;
    const float* const s = p.scores + (long long)g * p.prows * p.s_row + (long long)tile * TA_KEYS + 4 * lane;
    const float2* const stats = p.stats + (size_t)g * p.pad_rows;
    constexpr int AHEAD = 4;
    float4 x[AHEAD];
    float2 e[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
        const int r = first + k * groups;
        x[k] = r < rows ? __ldcg(reinterpret_cast<const float4*>(s + r * p.s_row)) : make_float4(0.f, 0.f, 0.f, 0.f);
        e[k] = !JOIN && r < rows ? __ldcg(stats + r) : make_float2(0.f, 0.f);
    }
    if constexpr (JOIN) {
#pragma unroll 1
        for (int r = warp; r < p.prows; r += WARPS) {
            float2 f[(TA_MAXSPLITS + 31) / 32];
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) {
                const int q = lane + 32 * k;
                f[k] = q < p.splits ? __ldcg(&p.part_ml[((size_t)q * p.kv_heads + g) * p.pad_rows + r]) : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) top = fmaxf(top, f[k].x);
#pragma unroll
            for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) sum += f[k].y * ex2(f[k].x - ref);
#pragma unroll
            for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            if (lane == 0) stat[r] = make_float2(ref, sum);
        }
        __syncthreads();
    }
    float a[4] = { 0.f, 0.f, 0.f, 0.f };
    auto add = [&](const float4& v, float2 st) {
        const float inv = st.y == 0.f ? 0.f : 1.f / st.y, s[4] = { v.x, v.y, v.z, v.w };
        // a masked slot's score is -inf: it gets nothing, be the row's sum NaN (0 * NaN)
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = s[i] == -INFINITY ? a[i] : fmaf(ex2(s[i] - st.x), inv, a[i]);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; k++) if (first + k * groups < rows) add(x[k], JOIN ? stat[first + k * groups] : e[k]);
#pragma unroll 4
    for (int r = first + AHEAD * groups; r < rows; r += groups) add(__ldcg(reinterpret_cast<const float4*>(s + r * p.s_row)), JOIN ? stat[r] : __ldcg(stats + r));
    store4(&part[warp][4 * lane], a);
    __syncthreads();
    for (int k = tid; k < WARPS / groups * TA_KEYS; k += 32 * WARPS) {
        const int w0 = k / TA_KEYS * groups, c = k % TA_KEYS;
        const long long slot = (long long)b * (WARPS / groups) * TA_KEYS + k;
        if (slot >= total) break;
        float sum = part[w0][c];
        for (int w = 1; w < groups; w++) sum += part[w0 + w][c];
        p.weights[g * p.w_head + slot] += sum;
    }
}

// Joins the runs of one product row: out = sum of the runs' outputs, each scaled to the common reference, over the sum of their sums, in a fixed order.  Four groups of
// HD / 4 threads take every fourth run; runs that saw nothing are not read.  Latency: the gate and the first outputs are asked for before the weights are known, and every
// warp forms the weights of all runs for itself instead of meeting the others.  CTAs behind the rows' form received weights.
template <class TA, int NB>
__global__ void __launch_bounds__(64 * NB) k_tree_join(const __grid_constant__ TaParams p) {
    constexpr int HD = 64 * NB, LANES = HD / 4, WARPS = 2 * NB, AHEAD = 4;
    __shared__ float wgt[WARPS][TA_MAXSPLITS];
    __shared__ float4 acc[3][LANES];
    const int tid = threadIdx.x, r = blockIdx.x, g = blockIdx.y, warp = tid >> 5, lane = tid & 31;
    if (r >= p.prows) {
        asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
        ta_weigh<WARPS, true>(p, r - p.prows, g, tid);
        return;
    }
    const int grp = tid / LANES, c = tid % LANES * 4;
    const int t = ta_row(p, r), h = g * p.group + r - t * p.group;
    float z[4] = { 0.f, 0.f, 0.f, 0.f };
    // The gate is the caller's: nothing in this call writes it, and the kernel before lets this one begin only when whatever wrote it has ended.
    if (p.gate && grp == 0 && c < p.dim) load4((const TA*)p.gate + t * p.g_row + h * p.g_head + c, z);
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const size_t step = (size_t)p.kv_heads * p.pad_rows, at = (size_t)g * p.pad_rows + r;
    const float* const o = p.part_o + at * HD + c;
    float2 e[(TA_MAXSPLITS + 31) / 32];
    float4 v[AHEAD];
#pragma unroll
    for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) { const int s = lane + 32 * k; e[k] = s < p.splits ? __ldcg(&p.part_ml[s * step + at]) : make_float2(-INFINITY, 0.f); }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) { const int s = grp + 4 * k; v[k] = s < p.splits ? __ldcg(reinterpret_cast<const float4*>(o + s * step * HD)) : make_float4(0.f, 0.f, 0.f, 0.f); }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) top = fmaxf(top, e[k].x);
#pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < (TA_MAXSPLITS + 31) / 32; k++) {
        const int s = lane + 32 * k;
        const float w = ex2(e[k].x - ref);
        if (s < p.splits) wgt[warp][s] = e[k].x == -INFINITY && e[k].y == 0.f ? -1.f : w;           // -1: saw nothing
        sum += e[k].y * w;
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    __syncwarp();
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, const float4& x) {
        if (w < 0.f) return;
        a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y); a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; k++) if (grp + 4 * k < p.splits) add(wgt[warp][grp + 4 * k], v[k]);
#pragma unroll 4
    for (int s = grp + 4 * AHEAD; s < p.splits; s += 4) add(wgt[warp][s], __ldcg(reinterpret_cast<const float4*>(o + s * step * HD)));
    if (grp) acc[grp - 1][tid % LANES] = a;
    __syncthreads();
    if (p.stats && tid == 0) p.stats[at] = make_float2(ref, sum);
    if (grp || c >= p.dim) return;
#pragma unroll
    for (int k = 0; k < 3; k++) { const float4 x = acc[k][tid]; a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w; }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    float out[4] = { a.x * inv, a.y * inv, a.z * inv, a.w * inv };
    if (p.gate) {
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] /= 1.f + __expf(-z[i]);
    }
    store4((TA*)p.out + t * p.o_row + h * p.o_head + c, out);
}

// The received weights of runs that have joined.
__global__ void __launch_bounds__(256) k_tree_weights(const __grid_constant__ TaParams p) {
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    ta_weigh<8, false>(p, blockIdx.x, blockIdx.y, threadIdx.x);
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
// How a call is cut: rows of a CTA's product tile, tiles of product rows, runs of the cache.
struct TaPlan { int nb, nr, pad_rows, row_tiles, splits; bool joined, scores; size_t part_o, part_ml, stats, kept, total; };

long ta_tiles(const it_tree_attention_args* a) { return ((long)a->cached + a->rows + TA_KEYS - 1) / TA_KEYS; }
TaPlan ta_plan(const it_tree_attention_args* a, const it_tree_cut& c) {
    TaPlan pl;
    pl.nb = a->head_dim <= 128 ? 2 : 4;
    pl.nr = c.nr; pl.row_tiles = c.row_tiles; pl.splits = c.splits; pl.joined = c.joined;
    pl.pad_rows = pl.row_tiles * pl.nr;
    const size_t splits = (size_t)pl.splits;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = (size_t)a->kv_heads * pl.pad_rows;
    pl.part_o = 0;
    pl.part_ml = !pl.joined ? up(splits * rows * 64 * pl.nb * 4) : 0;
    pl.stats = pl.part_ml + (!pl.joined ? up(splits * rows * 8) : 0);
    pl.kept = pl.stats + up(rows * 8);
    const size_t prows = (size_t)a->rows * (a->heads / a->kv_heads);
    pl.scores = a->weights && it_tree_keeps_scores((long)prows, a->kv_heads, a->head_dim, ta_tiles(a));
    pl.total = pl.kept + (pl.scores ? prows * a->kv_heads * ta_tiles(a) * TA_KEYS * 4 : 0);
    return pl;
}

typedef CUresult (*ta_encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int ta_map(CUtensorMap* map, const void* cache, int type, int dim, int64_t slots, int64_t slot, int heads, int64_t head) {
    static ta_encode_fn encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* fn = nullptr; cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) encode = (ta_encode_fn)fn;
    });
    if (!encode) return it_fail(IT_ECUDA, "it_tree_attention: the driver does not export cuTensorMapEncodeTiled");
    if (slots == 1) slot = dim;                // an axis of one: any stride will do
    if (heads == 1) head = dim;
    const cuuint64_t dims[3] = { (cuuint64_t)dim, (cuuint64_t)slots, (cuuint64_t)heads };
    const cuuint64_t strides[2] = { (cuuint64_t)slot * 2, (cuuint64_t)head * 2 };
    const cuuint32_t box[3] = { 64, TA_KEYS, 1 }, estr[3] = { 1, 1, 1 };
    const CUresult r = encode(map, type == IT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(cache), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? IT_OK : it_fail(IT_ECUDA, "it_tree_attention: cuTensorMapEncodeTiled failed with code %d", (int)r);
}

// Every kernel is loaded, and its shared memory allowed, by the first call on a device, so that later calls can be recorded.
int ta_prepare(int device) {
    static std::mutex lock; static bool done[64] = {};
    std::lock_guard<std::mutex> hold(lock);
    if (done[device]) return IT_OK;
    if (const int r = it_tree_tc_prepare()) return r;
    auto load = [](auto kern) -> int { cudaFuncAttributes at; IT_CUDA(cudaFuncGetAttributes(&at, kern)); return IT_OK; };
    for (const int r : { load(k_tree_join<float, 2>), load(k_tree_join<float, 4>), load(k_tree_join<__half, 2>), load(k_tree_join<__half, 4>), load(k_tree_join<__nv_bfloat16, 2>), load(k_tree_join<__nv_bfloat16, 4>), load(k_tree_weights) })
        if (r) return r;
    done[device] = true;
    return IT_OK;
}

// CTAs of `warps` warps that form received weights.  All warps of one share a tile, or, where there are many tiles, as many as have four rows each (one row at 30,000 slots: 33.5 us for the call
// with a tile a CTA and a kernel more, 29.3).
int ta_weigh_ctas(TaParams& p, int warps) {
    const int tiles = (p.cached + p.rows + TA_KEYS - 1) / TA_KEYS;
    p.tile_warps = warps;
    while (p.tile_warps > 1 && 4 * (p.tile_warps / 2) >= p.prows && (long)tiles * p.kv_heads > 2 * TA_MAXSPLITS) p.tile_warps /= 2;
    const int each = warps / p.tile_warps;
    return (tiles + each - 1) / each;
}
int ta_join(TaParams& p, int type, int nb, cudaStream_t st) {
    const int more = p.scores && p.prows <= TA_JOINROWS ? ta_weigh_ctas(p, 2 * nb) : 0;
    auto go = [&](auto kern) -> int { IT_CUDA(it_launch_early(kern, dim3(p.prows + more, p.kv_heads), dim3(64 * nb), 0, st, 1, p)); return IT_OK; };
    if (type == IT_F32) return nb == 2 ? go(k_tree_join<float, 2>) : go(k_tree_join<float, 4>);
    if (type == IT_F16) return nb == 2 ? go(k_tree_join<__half, 2>) : go(k_tree_join<__half, 4>);
    return nb == 2 ? go(k_tree_join<__nv_bfloat16, 2>) : go(k_tree_join<__nv_bfloat16, 4>);
}

int ta_check_sizes(const it_tree_attention_args* a) {
    const char* const who = "it_tree_attention";
    IT_CHECK_ARG(a, "%s: null argument", who);
    IT_CHECK_ARG(it_type_pair(a->type, a->cache_type), "%s: types %d over %d", who, a->type, a->cache_type);
    IT_CHECK_ARG(a->rows >= 0 && a->rows <= TA_MAXROWS, "%s: %d rows, at most %d", who, a->rows, TA_MAXROWS);
    IT_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, "%s: head dimension %d is not a multiple of 8 up to 256", who, a->head_dim);
    IT_CHECK_ARG(a->kv_heads >= 1 && a->kv_heads <= 4096 && a->heads >= 1 && a->heads % a->kv_heads == 0 && a->heads / a->kv_heads <= 1024, "%s: %d heads over %d kv heads", who, a->heads, a->kv_heads);
    IT_CHECK_ARG(a->cached >= 0 && a->cached < ((int64_t)1 << 30), "%s: %lld cached slots", who, (long long)a->cached);
    return IT_OK;
}

}  // namespace

IT_API int it_tree_attention_workspace(const it_tree_attention_args* a, size_t* nbytes) {
    if (const int r = ta_check_sizes(a)) return r;
    IT_CHECK_ARG(nbytes, "it_tree_attention_workspace: null argument");
    // the most that any cut of these sizes asks for: it then grows with `cached`, and a workspace for a long cache serves a shorter one, which may be cut another way
    *nbytes = 0;
    for (int nr = 16; a->rows && nr <= 64; nr *= 2) {
        const it_tree_cut c = it_tree_cut_by(nr, (long)a->rows * (a->heads / a->kv_heads), a->kv_heads, ta_tiles(a), TA_MAXSPLITS);
        const size_t n = ta_plan(a, c).total;
        if (n > *nbytes) *nbytes = n;
        if (c.row_tiles == 1) break;
    }
    const long prows = (long)a->rows * (a->heads / a->kv_heads);
    if (a->rows && a->weights && !it_tree_keeps_scores(prows, a->kv_heads, a->head_dim, ta_tiles(a))) *nbytes += IT_TREE_SCORE_BYTES;       // a shorter cache's would be kept
    return IT_OK;
}

IT_API int it_tree_attention(void* stream, const it_tree_attention_args* a) {
    const char* const who = "it_tree_attention";
    if (const int r = ta_check_sizes(a)) return r;
    if (a->rows == 0) return IT_OK;
    IT_CHECK_ARG(a->q && a->out && a->k_cache && a->v_cache, "%s: null pointer", who);
    const int64_t T = a->rows, H = a->heads, G = a->kv_heads, D = a->head_dim;
    const size_t es = it_type_size(a->type), al = 4 * es;
    IT_CHECK_ARG(a->slots >= 1 && a->slots < ((int64_t)1 << 31) && a->cached + T <= a->slots, "%s: %lld cached slots and %d rows in a cache of %lld", who, (long long)a->cached, a->rows, (long long)a->slots);
    IT_CHECK_ARG(it_aligned(a->q, al) && it_aligned(a->out, al) && it_aligned(a->gate, al) && it_strides_ok(T, a->q_row, H, a->q_head, D, 4) && it_strides_ok(T, a->o_row, H, a->o_head, D, 4) &&
                 (!a->gate || it_strides_ok(T, a->g_row, H, a->g_head, D, 4)), "%s: q, gate or out: pointers and strides are multiples of 4 elements, strides hold what lies between", who);
    IT_CHECK_ARG(it_aligned(a->k_cache, 16) && it_aligned(a->v_cache, 16) && it_strides_ok(a->slots, a->kc_slot, G, a->kc_head, D, 8) && it_strides_ok(a->slots, a->vc_slot, G, a->vc_head, D, 8),
                 "%s: caches: 16-byte aligned, strides are multiples of 8 elements and hold what lies between", who);
    IT_CHECK_ARG(it_aligned(a->parents, 4) && it_aligned(a->length, 4) && it_aligned(a->weights, 4), "%s: a pointer is not aligned to its type", who);
    IT_CHECK_ARG(!a->weights || G == 1 || a->w_head >= a->cached + T, "%s: weights of a head overlap the next one's", who);
    IT_CHECK_ARG(a->scale == a->scale && a->scale <= 3e38f && a->scale >= -3e38f, "%s: bad scale", who);
    const size_t os = it_span(T, a->o_row, H, a->o_head, D, es);
    auto same = [&](const void* x, int64_t row, int64_t head) { return x == a->out && (T < 2 || row == a->o_row) && (H < 2 || head == a->o_head); };
    // a second walk for the received weights reads q after out is written
    IT_CHECK_ARG((same(a->q, a->q_row, a->q_head) && !a->weights) || !it_overlap(a->q, it_span(T, a->q_row, H, a->q_head, D, es), a->out, os), "%s: out overlaps q", who);
    IT_CHECK_ARG(!a->gate || same(a->gate, a->g_row, a->g_head) || !it_overlap(a->gate, it_span(T, a->g_row, H, a->g_head, D, es), a->out, os), "%s: out overlaps gate", who);
    const TaPlan pl = ta_plan(a, it_tree_cut_of((long)a->rows * (a->heads / a->kv_heads), a->kv_heads, a->head_dim, ta_tiles(a), TA_MAXSPLITS));
    // what a call writes is none of what it reads or writes elsewhere (out may be q or gate, see above)
    const it_stretch all[] = { { "out", a->out, os }, { "weights", a->weights, ((size_t)(G - 1) * (size_t)a->w_head + (size_t)(a->cached + T)) * 4 }, { "the workspace", a->workspace, pl.total },
                               { "k_cache", a->k_cache, it_span(a->cached + T, a->kc_slot, G, a->kc_head, D, 2) }, { "v_cache", a->v_cache, it_span(a->cached + T, a->vc_slot, G, a->vc_head, D, 2) },
                               { "q", a->q, it_span(T, a->q_row, H, a->q_head, D, es) }, { "gate", a->gate, it_span(T, a->g_row, H, a->g_head, D, es) } };
    for (int i = 0; i < 3; i++)
        if (const char* x = it_overlaps(all[i], all + i + 1, i == 0 ? 4 : 6 - i)) return it_fail(IT_EINVAL, "%s: %s overlaps %s", who, all[i].name, x);
    it_ops_device dev;
    if (const int r = it_ops_current(stream, who, &dev)) return r;
    if (const int r = ta_prepare(dev.device)) return r;
    IT_CHECK_ARG(a->workspace && it_aligned(a->workspace, 256) && a->workspace_bytes >= pl.total, "%s: a workspace of %zu bytes, 256-byte aligned, is needed", who, pl.total);
    CUtensorMap km, vm;
    if (const int r = ta_map(&km, a->k_cache, a->cache_type, a->head_dim, a->cached + T, a->kc_slot, a->kv_heads, a->kc_head)) return r;
    if (const int r = ta_map(&vm, a->v_cache, a->cache_type, a->head_dim, a->cached + T, a->vc_slot, a->kv_heads, a->vc_head)) return r;
    TaParams p;
    char* ws = (char*)a->workspace;
    p.q = a->q; p.gate = a->gate; p.out = a->out; p.parents = a->parents; p.length = a->length; p.weights = a->weights;
    p.part_o = (float*)(ws + pl.part_o); p.part_ml = (float2*)(ws + pl.part_ml); p.stats = a->weights ? (float2*)(ws + pl.stats) : nullptr; p.scores = pl.scores ? (float*)(ws + pl.kept) : nullptr; p.status = dev.status_dev;
    p.q_row = a->q_row; p.q_head = a->q_head; p.g_row = a->g_row; p.g_head = a->g_head; p.o_row = a->o_row; p.o_head = a->o_head; p.w_head = a->w_head; p.s_row = (long long)ta_tiles(a) * TA_KEYS;
    p.rows = a->rows; p.heads = a->heads; p.group = a->heads / a->kv_heads; p.kv_heads = a->kv_heads; p.dim = a->head_dim; p.cached = (int)a->cached; p.splits = pl.splits;
    p.prows = a->rows * p.group; p.pad_rows = pl.pad_rows; p.joined = pl.joined; p.tile_warps = 8; p.group_inv = (unsigned)((0x100000000ull + p.group - 1) / p.group); p.scale = a->scale == 0.f ? 1.f / sqrtf((float)a->head_dim) : a->scale;
    const cudaStream_t st = (cudaStream_t)stream;
    if (const int r = it_tree_tc_run(p, a->type, pl.nb, pl.nr, pl.row_tiles, km, vm, st)) return r;
    if (!p.joined) if (const int r = ta_join(p, a->type, pl.nb, st)) return r;
    if (p.scores) {
        const int ctas = ta_weigh_ctas(p, 8);
        if (p.joined || p.prows > TA_JOINROWS) IT_CUDA(it_launch_early(k_tree_weights, dim3(ctas, p.kv_heads), dim3(256), 0, st, 1, p));
        return IT_OK;
    }
    return p.weights ? it_tree_tc_weigh(p, a->type, pl.nb, km, st) : IT_OK;
}
