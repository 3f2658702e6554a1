// Eviction from a KV cache by received attention weight.  The reference's cache only grows (src/vk/mod.rs:765 asserts that it fits).
//
// Per KV head: the last `recent` slots stay, and of the others the keep - recent with the largest weight, ties to the lower slot; what stays moves to the front in
// its old order, in place.
//
// k_evict_select: weights as unsigned keys of the same order (NaN lowest), the smallest kept key by a radix search of 11 + 11 + 10 bits, then the kept slots in
// order.  A cluster of CTAs has a head (one CTA for short caches): each takes a run of slots, the histograms are summed through distributed shared memory.
// k_evict_move: the destination of a row is never behind its source and both are in order, so a CTA that walks all rows of ITS 16 or 32 bytes of a head front to back,
// reading a block of rows before it writes that block, never overwrites what it still has to read; nothing else touches those bytes.  Splitting a head by
// bytes instead of rows is what lets the copy run in place and in parallel.
#include "it_ops.cuh"
#include <cooperative_groups.h>
#include <mutex>
namespace cg = cooperative_groups;

namespace {

constexpr int EV_CLUSTER = 8, EV_THREADS = 512, EV_BINS = 2048;
constexpr int EV_MOVE_THREADS = 256, EV_UNROLL = 8;

struct EvParams {
    char *k, *v; float* weights; int* kept;
    long long kc_slot, kc_head, vc_slot, vc_head, w_head, kept_head;    // strides of the caches in bytes
    int kv_heads, n, keep, recent, row_bytes, slices, slice_bytes;
};

// An unsigned key in the order of the weights: -0 as 0, NaN below everything.
__device__ __forceinline__ unsigned ev_key(float w) {
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w == 0.f ? 0.f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int CL>
__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const __grid_constant__ EvParams p) {
    __shared__ unsigned hist[EV_BINS];
    __shared__ unsigned scan[EV_THREADS / 32], found[2], counts[2], warp_gt[EV_THREADS / 32], warp_eq[EV_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = CL > 1 ? (int)cluster.block_rank() : 0, g = blockIdx.x / CL;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* w = p.weights + (long long)g * p.w_head;
    int* kept = p.kept + (long long)g * p.kept_head;
    const int cand = p.n - p.recent, want = p.keep - p.recent;
    const int per = (cand + CL - 1) / CL, begin = min(cand, rank * per), end = min(cand, begin + per);
    for (int i = rank * EV_THREADS + tid; i < p.recent; i += CL * EV_THREADS) kept[want + i] = cand + i;
    if (want == 0) return;                     // every CTA of the cluster leaves here
    // ---- the smallest kept key, 11 + 11 + 10 bits; `left`: how many of the keys with the bits found so far are kept
    unsigned prefix = 0, left = (unsigned)want;
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int b = tid; b < EV_BINS; b += EV_THREADS) hist[b] = 0;
        __syncthreads();
        const unsigned above = pass == 0 ? 0 : prefix >> (shift + (pass == 2 ? 10 : 11));
#pragma unroll 8
        for (int i = begin + tid; i < end; i += EV_THREADS) {
            const unsigned key = ev_key(__ldg(w + i));
            if (pass == 0 || key >> (pass == 1 ? 21 : 10) == above) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        if (CL > 1) cluster.sync(); else __syncthreads();
        // four bins a thread, the highest first, summed over the cluster; a scan finds the bin in which the count reaches `left`
        unsigned c[4], sum = 0;
        const int top = bins - 1 - 4 * tid;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            c[j] = 0;
            if (top - j >= 0) {
                if (CL > 1) { for (int r = 0; r < CL; r++) c[j] += *cluster.map_shared_rank(&hist[top - j], r); }
                else c[j] = hist[top - j];
            }
            sum += c[j];
        }
        unsigned inc = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const unsigned o = __shfl_up_sync(0xffffffffu, inc, d); if (lane >= d) inc += o; }
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        unsigned before = inc - sum;
        for (int k = 0; k < warp; k++) before += scan[k];
        if (before < left && before + sum >= left) {          // one thread
            unsigned b = before; int j = 0;
            while (b + c[j] < left) b += c[j++];
            found[0] = (unsigned)(top - j); found[1] = left - b;
        }
        __syncthreads();
        prefix |= found[0] << shift; left = found[1];
        if (CL > 1) cluster.sync(); else __syncthreads();     // every CTA has read the histograms
    }
    // ---- kept: keys above `prefix`, and the first `left` of those equal to it, in slot order.  A warp has a run of its CTA's slots.
    const int wper = (end - begin + EV_THREADS / 32 - 1) / (EV_THREADS / 32), wb = min(end, begin + warp * wper), we = min(end, wb + wper);
    unsigned gt = 0, eq = 0;
#pragma unroll 4
    for (int i = wb; i < we; i += 32) {
        const unsigned key = i + lane < we ? ev_key(__ldg(w + i + lane)) : 0u;
        const bool in = i + lane < we;
        gt += __popc(__ballot_sync(0xffffffffu, in && key > prefix));
        eq += __popc(__ballot_sync(0xffffffffu, in && key == prefix));
    }
    if (lane == 0) { warp_gt[warp] = gt; warp_eq[warp] = eq; }
    __syncthreads();
    if (tid < 2) { unsigned s = 0; const unsigned* q = tid ? warp_eq : warp_gt; for (int k = 0; k < EV_THREADS / 32; k++) s += q[k]; counts[tid] = s; }
    if (CL > 1) cluster.sync(); else __syncthreads();
    unsigned gt0 = 0, eq0 = 0;
    for (int r = 0; r < rank; r++) { gt0 += *cluster.map_shared_rank(&counts[0], r); eq0 += *cluster.map_shared_rank(&counts[1], r); }
    for (int k = 0; k < warp; k++) { gt0 += warp_gt[k]; eq0 += warp_eq[k]; }
    const unsigned below = (1u << lane) - 1u;
#pragma unroll 4
    for (int i = wb; i < we; i += 32) {
        const bool in = i + lane < we;
        const unsigned key = in ? ev_key(__ldg(w + i + lane)) : 0u;
        const unsigned bg = __ballot_sync(0xffffffffu, in && key > prefix), be = __ballot_sync(0xffffffffu, in && key == prefix);
        const unsigned e = eq0 + __popc(be & below);
        const bool take = in && (key > prefix || (key == prefix && e < left));
        if (take) kept[gt0 + __popc(bg & below) + min(e, left)] = i + lane;
        gt0 += __popc(bg); eq0 += __popc(be);
    }
    if (CL > 1) cluster.sync();                // nobody leaves while its counts may still be read
}

// Rows front to back in blocks: a block is read by all threads before any of them writes it.  U: what one thread moves of a row.
template <class U>
__device__ void ev_move(char* base, long long stride, const int* kept, int keep, int lanes) {
    const int tid = threadIdx.x, rows = EV_MOVE_THREADS / lanes, r = tid / lanes, x = tid % lanes * (int)sizeof(U);
    for (int b = 0; b < keep; b += rows * EV_UNROLL) {
        U v[EV_UNROLL]; bool go[EV_UNROLL];
#pragma unroll
        for (int j = 0; j < EV_UNROLL; j++) {
            const int i = b + j * rows + r, s = i < keep ? __ldcg(kept + i) : 0;
            go[j] = i < keep && s != i;
            if (go[j]) v[j] = __ldcg(reinterpret_cast<const U*>(base + s * stride + x));
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EV_UNROLL; j++) if (go[j]) *reinterpret_cast<U*>(base + (b + j * rows + r) * stride + x) = v[j];
    }
}
__global__ void __launch_bounds__(EV_MOVE_THREADS) k_evict_move(const __grid_constant__ EvParams p) {
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const int g = blockIdx.y, job = blockIdx.x;
    const int* kept = p.kept + (long long)g * p.kept_head;
    if (job == 2 * p.slices) { ev_move<float>((char*)(p.weights + (long long)g * p.w_head), 4, kept, p.keep, 1); return; }
    const bool is_v = job >= p.slices;
    char* c = is_v ? p.v : p.k;
    if (!c) return;
    const int s = is_v ? job - p.slices : job;
    ev_move<uint4>(c + (long long)g * (is_v ? p.vc_head : p.kc_head) + s * p.slice_bytes, is_v ? p.vc_slot : p.kc_slot, kept, p.keep, p.slice_bytes / 16);
}

int ev_check_sizes(const it_cache_evict_args* a) {
    const char* const who = "it_cache_evict";
    IT_CHECK_ARG(a, "%s: null argument", who);
    IT_CHECK_ARG(a->kv_heads >= 1 && a->kv_heads <= 4096, "%s: %d kv heads", who, a->kv_heads);
    IT_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, "%s: head dimension %d is not a multiple of 8 up to 256", who, a->head_dim);
    IT_CHECK_ARG(a->recent >= 0 && a->recent <= a->keep && a->keep <= a->n && a->n <= a->slots && a->n <= (1 << 20), "%s: keep %lld, the last %lld of them, of %lld slots in a cache of %lld", who,
                 (long long)a->keep, (long long)a->recent, (long long)a->n, (long long)a->slots);
    return IT_OK;
}

}  // namespace

IT_API int it_cache_evict_workspace(const it_cache_evict_args* a, size_t* nbytes) {
    if (const int r = ev_check_sizes(a)) return r;
    IT_CHECK_ARG(nbytes, "it_cache_evict_workspace: null argument");
    *nbytes = a->kept ? 0 : ((size_t)a->kv_heads * a->keep * 4 + 255) / 256 * 256;
    return IT_OK;
}

IT_API int it_cache_evict(void* stream, const it_cache_evict_args* a) {
    const char* const who = "it_cache_evict";
    size_t need = 0;
    if (const int r = it_cache_evict_workspace(a, &need)) return r;
    if (a->keep == 0) return IT_OK;
    const int64_t G = a->kv_heads, D = a->head_dim;
    IT_CHECK_ARG(a->weights && it_aligned(a->weights, 4) && (G == 1 || a->w_head >= a->n), "%s: weights are given, and a head's do not overlap the next one's", who);
    IT_CHECK_ARG(it_aligned(a->k_cache, 16) && it_aligned(a->v_cache, 16) && (!a->k_cache || it_strides_ok(a->slots, a->kc_slot, G, a->kc_head, D, 8)) &&
                 (!a->v_cache || it_strides_ok(a->slots, a->vc_slot, G, a->vc_head, D, 8)), "%s: caches: 16-byte aligned, strides are multiples of 8 elements and hold what lies between", who);
    IT_CHECK_ARG(!a->kept || (it_aligned(a->kept, 4) && (G == 1 || a->kept_head >= a->keep)), "%s: kept: a head's slots do not overlap the next one's", who);
    IT_CHECK_ARG(need == 0 || (a->workspace && it_aligned(a->workspace, 256) && a->workspace_bytes >= need), "%s: a workspace of %zu bytes, 256-byte aligned, is needed", who, need);
    it_ops_device dev;
    if (const int r = it_ops_current(stream, who, &dev)) return r;
    static std::mutex lock; static bool loaded[64] = {};
    {
        std::lock_guard<std::mutex> hold(lock);
        if (!loaded[dev.device]) {             // the kernels are loaded by the first call, so that later ones can be recorded
            cudaFuncAttributes at;
            IT_CUDA(cudaFuncGetAttributes(&at, k_evict_select<1>));
            IT_CUDA(cudaFuncGetAttributes(&at, k_evict_select<EV_CLUSTER>));
            IT_CUDA(cudaFuncGetAttributes(&at, k_evict_move));
            loaded[dev.device] = true;
        }
    }
    EvParams p;
    p.k = (char*)a->k_cache; p.v = (char*)a->v_cache; p.weights = a->weights; p.kept = a->kept ? a->kept : (int*)a->workspace;
    p.kc_slot = a->kc_slot * 2; p.kc_head = a->kc_head * 2; p.vc_slot = a->vc_slot * 2; p.vc_head = a->vc_head * 2; p.w_head = a->w_head; p.kept_head = a->kept ? a->kept_head : a->keep;
    p.kv_heads = a->kv_heads; p.n = (int)a->n; p.keep = (int)a->keep; p.recent = (int)a->recent; p.row_bytes = a->head_dim * 2;
    // 32 bytes a row and CTA, a memory sector; 16 where a head is not a multiple of that or the CTAs would not fill the GPU
    p.slice_bytes = p.row_bytes % 32 || (long)p.row_bytes / 32 * 2 * a->kv_heads < dev.sm_count / 2 ? 16 : 32;
    p.slices = p.row_bytes / p.slice_bytes;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const bool wide = p.n - p.recent > 8192;
    cfg.gridDim = dim3((unsigned)(a->kv_heads * (wide ? EV_CLUSTER : 1))); cfg.blockDim = dim3(EV_THREADS); cfg.stream = st; cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = EV_CLUSTER; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = wide ? 1 : 0;
    if (wide) IT_CUDA(cudaLaunchKernelEx(&cfg, k_evict_select<EV_CLUSTER>, p));
    else IT_CUDA(cudaLaunchKernelEx(&cfg, k_evict_select<1>, p));
    cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * p.slices + 1), (unsigned)a->kv_heads); cfg.blockDim = dim3(EV_MOVE_THREADS); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    IT_CUDA(cudaLaunchKernelEx(&cfg, k_evict_move, p));
    return IT_OK;
}
