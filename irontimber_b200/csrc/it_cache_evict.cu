// Eviction from a KV cache by received attention weight.  The reference's cache only grows (src/vk/mod.rs:765 asserts that it fits).
//
// Per KV head: the last `recent` slots stay, and of the others the keep - recent with the largest weight, ties to the lower slot; what stays moves to the front in
// its old order, in place.
//
// k_evict_select: a cluster of CTAs has a head (one CTA for short caches) and holds its weights in shared memory: one read for all passes.  The smallest kept weight is looked for
// from the top: a histogram over 2048 bins spread where such weights lie finds the bin that holds it, and the few weights of that bin are brought together and ranked; only where
// they are many, or lie outside, does the search go on 11 bits at a time (unsigned keys in the weights' order, NaN lowest).  Every CTA sums its share of a histogram's bins over the
// cluster and hands the sums out (reading all histograms from every CTA took 12 us a pass).  Three passes of 11 bits for all took 5.1 / 11.0 / 20.8 us at 1200 / 8192 / 131,072
// slots of 4 heads, this 4.3 / 8.6 / 19.9.  Then ballots give every kept slot its place, in order; the weights move here.
// k_evict_move: rows of a head are whole runs of memory, blocks of 64 of them a CTA.  In place, a block's destination may hold rows that others still have to read; kept slots are in order
// and never before their place, so those are rows of at most two earlier blocks (the select kernel notes how many kept slots lie before every 64th).  A block reads its
// rows into shared memory, says so, waits for those two, and writes.  Blocks are numbered as they start, so whom a block waits for has started before it.
#include "it_ops.cuh"
#include "it_ops_sites.h"
#include "it_pipe.cuh"
#include <cooperative_groups.h>
#include <mutex>
namespace cg = cooperative_groups;

namespace {

constexpr int EV_THREADS = 1024, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048, EV_BLOCK = 64, EV_MOVE_THREADS = 256, EV_CAND = EV_THREADS, EV_RANK = 128;
constexpr int EV_UNIT = EV_WARPS * EV_BLOCK, EV_PER = 32 * 32 * EV_WARPS;          // slots of a CTA are a multiple of the first (every warp has whole blocks) and at most the second (a lane for every 32 of a warp's)

struct EvParams {
    char *k, *v; float* weights; int *kept, *ranks, *status; unsigned *flags;       // flags: [0] blocks started, then one per block: its rows are read
    long long kc_slot, kc_head, vc_slot, vc_head, w_head, kept_head;                // strides of the caches in bytes
    int kv_heads, n, keep, recent, row_bytes, per, rank_head, blocks, nflags;
};

// An unsigned key in the order of the weights: -0 as 0, NaN below everything.
__device__ __forceinline__ unsigned ev_key(float w) {
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w == 0.f ? 0.f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A first histogram's bin, in the keys' order: 64 an octave of the weights from 2^-22 to 2^10, where received attention lies, everything else in the outer two.  The keys' own upper bits
// give four an octave, in which a warp's additions meet.
constexpr int EV_SHIFT = 17;
constexpr unsigned EV_FIRST = (0x80000000u >> EV_SHIFT) + ((127 - 22) << (23 - EV_SHIFT)) - 1;      // bin 0 ends with it
__device__ __forceinline__ unsigned ev_bin(unsigned key) { return (unsigned)min(max((int)(key >> EV_SHIFT) - (int)EV_FIRST, 0), EV_BINS - 1); }

template <int CL>
__global__ void __launch_bounds__(EV_THREADS, 1) k_evict_select(const __grid_constant__ EvParams p) {
    extern __shared__ float w_s[];                     // [per]
    __shared__ unsigned hist[EV_BINS], total[EV_BINS];
    __shared__ unsigned mine[EV_CAND], all[EV_CAND], few[EV_RANK];
    __shared__ unsigned scan[EV_WARPS], found[4], warp_gt[EV_WARPS], warp_eq[EV_WARPS], counts[2], nmine, nfew;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = CL > 1 ? (int)cluster.block_rank() : 0, g = blockIdx.x / CL;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto sync = [&] { if (CL > 1) cluster.sync(); else __syncthreads(); };
    float* w = p.weights + (long long)g * p.w_head;
    int* kept = p.kept + (long long)g * p.kept_head;
    int* ranks = p.ranks + (long long)g * p.rank_head;
    const int cand = p.n - p.recent, want = p.keep - p.recent;
    const int begin = rank * p.per, len = max(0, min(p.n - begin, p.per)), clen = max(0, min(cand - begin, p.per));      // this CTA's slots, and those of them that compete
    hist[tid] = 0; hist[tid + EV_THREADS] = 0;
    if (tid == 0) nmine = nfew = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = blockIdx.x * EV_THREADS + tid; i < p.nflags; i += gridDim.x * EV_THREADS) p.flags[i] = 0u;
#pragma unroll 8
    for (int i = tid; i < (len + 31) / 32 * 32; i += EV_THREADS) {
        const float x = i < len ? w[begin + i] : 0.f;
        const unsigned bin = ev_bin(ev_key(x)), low = __ballot_sync(0xffffffffu, i < clen && bin == 0);      // the slots that nothing looks at, in one addition
        if (i < len) w_s[i] = x;
        if (i < clen && bin > 0) atomicAdd(&hist[bin], 1u);
        if (lane == 0 && low) atomicAdd(&hist[0], (unsigned)__popc(low));
    }
    sync();                                            // every weight is read before any is written
    // ---- the smallest kept key: keys whose bits from `shift` up are `prefix` hold it, `count` of them, of which the `left` largest are kept
    unsigned prefix = want ? 0u : 0xffffffffu, left = (unsigned)want;
    if (want) {
        int shift = 32, bins = EV_BINS;
        bool spread = true;
#pragma unroll 1
        while (true) {
            // the bin in which the count from the top reaches `left`
            const unsigned* sums = hist;
            if (CL > 1) {
                constexpr int SHARE = EV_BINS / CL;
                if (tid < SHARE) {
                    const int b = rank * SHARE + tid;
                    unsigned c[CL], s = 0;
#pragma unroll
                    for (int r = 0; r < CL; r++) c[r] = *cluster.map_shared_rank(&hist[b], r);
#pragma unroll
                    for (int r = 0; r < CL; r++) s += c[r];
#pragma unroll
                    for (int r = 0; r < CL; r++) *cluster.map_shared_rank(&total[b], r) = s;
                }
                sync();
                sums = total;
            }
            // two bins a thread, the highest first
            const int top = bins - 1 - 2 * tid;
            const unsigned c0 = top >= 0 ? sums[top] : 0u, c1 = top >= 1 ? sums[top - 1] : 0u, sum = c0 + c1;
            unsigned inc = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const unsigned o = __shfl_up_sync(0xffffffffu, inc, d); if (lane >= d) inc += o; }
            if (lane == 31) scan[warp] = inc;
            __syncthreads();
            const unsigned before = inc - sum + __reduce_add_sync(0xffffffffu, lane < warp ? scan[lane] : 0u);
            if (before < left && before + sum >= left) {          // one thread
                const bool first = before + c0 >= left;
                found[0] = (unsigned)(first ? top : top - 1); found[1] = left - (first ? before : before + c0); found[2] = first ? c0 : c1;
            }
            __syncthreads();
            const unsigned bin = found[0], count = found[2];
            if (!spread) { prefix = prefix << (31 - __clz(bins)) | bin; left = found[1]; shift -= 31 - __clz(bins); }
            else if (bin > 0 && bin < EV_BINS - 1) { prefix = EV_FIRST + bin; left = found[1]; shift = EV_SHIFT; }
            const bool open = shift == 32;                          // an outer bin: nothing is known, from the start with the keys' own bits
            spread = false;
            if (shift == 0) break;
            if (!open && count <= EV_CAND) {
                // few enough for one a thread: bit by bit, each a count over the block, down to EV_RANK of them, then everyone's place among those (17 counts: 2.4 us)
#pragma unroll 8
                for (int i = tid; i < clen; i += EV_THREADS) {
                    const unsigned key = ev_key(w_s[i]);
                    if (key >> shift == prefix) mine[atomicAdd(&nmine, 1u)] = key;
                }
                sync();
                const unsigned* list = mine;
                if (CL > 1) {
                    if (warp < CL) {
                        const unsigned nr = lane < CL ? *cluster.map_shared_rank(&nmine, lane) : 0u, at = __reduce_add_sync(0xffffffffu, lane < warp ? nr : 0u), n = __shfl_sync(0xffffffffu, nr, warp);
                        const unsigned* from = cluster.map_shared_rank(mine, warp);
                        for (unsigned i = lane; i < n; i += 32) all[at + i] = from[i];
                    }
                    __syncthreads();
                    list = all;
                }
                bool in = tid < (int)count;
                unsigned key = in ? list[tid] : 0u;
                unsigned n = count, bit = 1u << (shift - 1);
                prefix <<= shift;
                for (; n > EV_RANK && bit; bit >>= 1) {
                    const unsigned set = (unsigned)__syncthreads_count(in && (key & bit)), up = set >= left;
                    if (up) prefix |= bit; else left -= set;
                    n = up ? set : n - set;
                    in = in && ((key & bit) != 0) == up;
                }
                if (bit) {                                          // (else all of them are equal)
                    if (n < count) {
                        if (in) few[atomicAdd(&nfew, 1u)] = key;
                        __syncthreads();
                        list = few;
                        if (tid < (int)n) key = few[tid];
                    }
                    if (tid < (int)n) {                             // the first warps only
                        unsigned more = 0, same = 0;
#pragma unroll 16
                        for (unsigned i = 0; i < n; i++) { const unsigned o = list[i]; more += o > key; same += o == key; }
                        if (more < left && more + same >= left) { found[0] = key; found[3] = left - more; }          // equal keys write equal values
                    }
                    __syncthreads();
                    prefix = found[0]; left = found[3];
                }
                break;
            }
            // the next eleven bits, or the last ones, of the keys that have these
            const int bits = shift > 11 ? 11 : shift, down = shift - bits;
            bins = 1 << bits;
            sync();                                                 // everyone has read the sums before
            hist[tid] = 0; hist[tid + EV_THREADS] = 0;
            __syncthreads();
#pragma unroll 8
            for (int i = tid; i < clen; i += EV_THREADS) {
                const unsigned key = ev_key(w_s[i]);
                if (open || key >> shift == prefix) atomicAdd(&hist[(key >> down) & (bins - 1)], 1u);
            }
            sync();
        }
    }
    // ---- kept: the last slots, keys above `prefix`, and the first `left` of those equal to it, in slot order.  A warp has a run of its CTA's slots.
    const int wper = p.per / EV_WARPS, wb = warp * wper, we = min(len, wb + wper);
    unsigned gt = 0, eq = 0, is_gt = 0, is_eq = 0;             // is_*: of the run's `lane`th 32 slots
#pragma unroll 4
    for (int i = wb; i < we; i += 32) {
        const bool in = i + lane < we;
        const unsigned key = in ? ev_key(w_s[i + lane]) : 0u;
        const bool last = begin + i + lane >= cand;
        const unsigned bg = __ballot_sync(0xffffffffu, in && (last || key > prefix)), be = __ballot_sync(0xffffffffu, in && !last && key == prefix);
        if (lane == (i - wb) / 32) { is_gt = bg; is_eq = be; }
        gt += __popc(bg); eq += __popc(be);
    }
    if (lane == 0) { warp_gt[warp] = gt; warp_eq[warp] = eq; }
    __syncthreads();
    if (warp == 0) {
        const unsigned a = __reduce_add_sync(0xffffffffu, warp_gt[lane]), b = __reduce_add_sync(0xffffffffu, warp_eq[lane]);
        if (lane == 0) { counts[0] = a; counts[1] = b; }
    }
    sync();
    unsigned a = lane < warp ? warp_gt[lane] : 0u, b = lane < warp ? warp_eq[lane] : 0u;
    if (CL > 1 && lane < rank) { a += *cluster.map_shared_rank(&counts[0], lane); b += *cluster.map_shared_rank(&counts[1], lane); }
    unsigned gt0 = __reduce_add_sync(0xffffffffu, a), eq0 = __reduce_add_sync(0xffffffffu, b);
    const unsigned below = (1u << lane) - 1u;
#pragma unroll 4
    for (int i = wb; i < we; i += 32) {
        const unsigned bg = __shfl_sync(0xffffffffu, is_gt, (i - wb) / 32), be = __shfl_sync(0xffffffffu, is_eq, (i - wb) / 32);
        if (lane == 0 && i % EV_BLOCK == 0) ranks[(begin + i) / EV_BLOCK] = (int)(gt0 + min(eq0, left));
        const unsigned e = eq0 + __popc(be & below);
        if ((bg >> lane & 1u) || ((be >> lane & 1u) && e < left)) {
            const unsigned at = gt0 + __popc(bg & below) + min(e, left);
            kept[at] = begin + i + lane; w[at] = w_s[i + lane];
        }
        gt0 += __popc(bg); eq0 += __popc(be);
    }
    if (rank == 0 && tid == 0) ranks[(p.n + EV_BLOCK - 1) / EV_BLOCK] = p.keep;
    if (CL > 1) cluster.sync();                // nobody leaves while its counts may still be read
}

__global__ void __launch_bounds__(EV_MOVE_THREADS) k_evict_move(const __grid_constant__ EvParams p) {
    extern __shared__ __align__(16) unsigned char rows[];          // [64][row_bytes]
    __shared__ int src[EV_BLOCK];
    __shared__ unsigned turn;
    __shared__ int go;
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    if (tid == 0) turn = atomicAdd(p.flags, 1u);
    __syncthreads();
    // block by block over all heads and both caches: whoever a block waits for has a lower number
    const int lines = p.kv_heads * ((p.k != nullptr) + (p.v != nullptr)), b = (int)turn / lines, line = (int)turn % lines, g = line % p.kv_heads;
    const bool is_v = line >= p.kv_heads || !p.k;
    char* const base = is_v ? p.v + (long long)g * p.vc_head : p.k + (long long)g * p.kc_head;
    const long long stride = is_v ? p.vc_slot : p.kc_slot;
    const int r0 = b * EV_BLOCK, nr = min(EV_BLOCK, p.keep - r0);
    const int* kept = p.kept + (long long)g * p.kept_head + r0;
    unsigned* const flags = p.flags + 1 + (size_t)line * p.blocks;
    const int* ranks = p.ranks + (long long)g * p.rank_head;
    if (tid < nr) src[tid] = __ldcg(kept + tid);
    __syncthreads();
    if (src[nr - 1] == r0 + nr - 1) {           // nothing moves up to here: nobody waits for rows that stay
        return;
    }
    const int pieces = p.row_bytes / 16;
#pragma unroll 8
    for (int i = tid; i < nr * pieces; i += EV_MOVE_THREADS) {
        const int r = i / pieces, c = i - r * pieces;
        cp_async16(rows + (size_t)i * 16, base + src[r] * stride + c * 16);
    }
    cp_async_wait_all();
    __syncthreads();
    if (tid == 0) {
        // this block's rows are read (the copies above are complete); then for the blocks whose rows lie where this one's go
        asm volatile("st.release.gpu.global.u32 [%0], %1;" :: "l"(flags + b), "r"(1u) : "memory");
        const int i0 = __ldcg(ranks + b), i1 = __ldcg(ranks + b + 1), q0 = i0 / EV_BLOCK, q1 = min(b, (i1 + EV_BLOCK - 1) / EV_BLOCK);
        const long long t0 = clock64();
        int ok = 1;
        for (int q = q0; q < q1; q++) {
            unsigned seen = 0;
            while (true) {
                asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(flags + q) : "memory");
                if (seen) break;
                if (clock64() - t0 > WAIT_CLOCKS) { atomicExch(p.status, IT_SITE_EVICT_MOVE); ok = 0; break; }
            }
            if (!ok) break;
        }
        go = ok;
    }
    __syncthreads();
    if (!go) return;
#pragma unroll 8
    for (int i = tid; i < nr * pieces; i += EV_MOVE_THREADS) {
        const int r = i / pieces, c = i - r * pieces;
        if (src[r] != r0 + r) *reinterpret_cast<uint4*>(base + (r0 + r) * stride + c * 16) = *reinterpret_cast<const uint4*>(rows + (size_t)i * 16);
    }
}

// Parts of a call's workspace, and how the weights are cut.
struct EvPlan { int cluster, per, rank_head, blocks; size_t kept, ranks, flags, nflags, total; };
EvPlan ev_plan(const it_cache_evict_args* a) {
    EvPlan pl;
    // us of the selection, 4 heads, with 1 / 8 / 16 CTAs a head: 1200 slots 4.3 / 7.2 / 11.0, 4096 7.7 / 8.5 / 12.0, 8192 11.0 / 8.6 / 12.2, 32,768 34.0 / 11.5 / 13.8,
    // 65,536 - / 15.5 / 16.2, 131,072 - / 23.4 / 19.9, 262,144 - / 39.8 / 28.1
    pl.cluster = a->n <= 5120 ? 1 : a->n <= 81920 ? 8 : 16;
    pl.per = (int)(((a->n + pl.cluster - 1) / pl.cluster + EV_UNIT - 1) / EV_UNIT * EV_UNIT);
    pl.rank_head = (int)((a->n + EV_BLOCK - 1) / EV_BLOCK + 1);
    pl.blocks = (int)((a->keep + EV_BLOCK - 1) / EV_BLOCK);
    pl.nflags = (size_t)2 * a->kv_heads * pl.blocks + 1;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    pl.ranks = 0;
    pl.flags = up((size_t)a->kv_heads * pl.rank_head * 4);
    pl.kept = pl.flags + up(pl.nflags * 4);
    pl.total = pl.kept + up((size_t)a->kv_heads * a->keep * 4);
    return pl;
}

int ev_check_sizes(const it_cache_evict_args* a) {
    const char* const who = "it_cache_evict";
    IT_CHECK_ARG(a, "%s: null argument", who);
    IT_CHECK_ARG(a->kv_heads >= 1 && a->kv_heads <= 4096, "%s: %d kv heads", who, a->kv_heads);
    IT_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, "%s: head dimension %d is not a multiple of 8 up to 256", who, a->head_dim);
    IT_CHECK_ARG(a->recent >= 0 && a->recent <= a->keep && a->keep <= a->n && a->n <= a->slots && a->n <= (1 << 19), "%s: keep %lld, the last %lld of them, of %lld slots in a cache of %lld", who,
                 (long long)a->keep, (long long)a->recent, (long long)a->n, (long long)a->slots);
    return IT_OK;
}

template <int CL> int ev_prepare_select() {
    IT_CUDA(cudaFuncSetAttribute(k_evict_select<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_PER * 4));
    if (CL > 8) IT_CUDA(cudaFuncSetAttribute(k_evict_select<CL>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return IT_OK;
}
// The kernels are loaded by the first call on a device, so that later ones can be recorded.
int ev_prepare(int device) {
    static std::mutex lock; static bool done[64] = {};
    std::lock_guard<std::mutex> hold(lock);
    if (done[device]) return IT_OK;
    if (const int r = ev_prepare_select<1>()) return r;
    if (const int r = ev_prepare_select<8>()) return r;
    if (const int r = ev_prepare_select<16>()) return r;
    cudaFuncAttributes at;
    IT_CUDA(cudaFuncGetAttributes(&at, k_evict_move));
    done[device] = true;
    return IT_OK;
}
template <int CL> int ev_select(const EvParams& p, cudaStream_t st) {
    IT_CUDA(it_launch_early(k_evict_select<CL>, dim3((unsigned)(p.kv_heads * CL)), dim3(EV_THREADS), (size_t)p.per * 4, st, CL, p));
    return IT_OK;
}

}  // namespace

IT_API int it_cache_evict_workspace(const it_cache_evict_args* a, size_t* nbytes) {
    if (const int r = ev_check_sizes(a)) return r;
    IT_CHECK_ARG(nbytes, "it_cache_evict_workspace: null argument");
    *nbytes = a->keep ? ev_plan(a).total : 0;
    return IT_OK;
}

IT_API int it_cache_evict(void* stream, const it_cache_evict_args* a) {
    const char* const who = "it_cache_evict";
    if (const int r = ev_check_sizes(a)) return r;
    if (a->keep == 0) return IT_OK;
    const int64_t G = a->kv_heads, D = a->head_dim;
    IT_CHECK_ARG(a->weights && it_aligned(a->weights, 4) && (G == 1 || a->w_head >= a->n), "%s: weights are given, and a head's do not overlap the next one's", who);
    IT_CHECK_ARG(it_aligned(a->k_cache, 16) && it_aligned(a->v_cache, 16) && (!a->k_cache || it_strides_ok(a->slots, a->kc_slot, G, a->kc_head, D, 8)) &&
                 (!a->v_cache || it_strides_ok(a->slots, a->vc_slot, G, a->vc_head, D, 8)), "%s: caches: 16-byte aligned, strides are multiples of 8 elements and hold what lies between", who);
    IT_CHECK_ARG(!a->kept || (it_aligned(a->kept, 4) && (G == 1 || a->kept_head >= a->keep)), "%s: kept: a head's slots do not overlap the next one's", who);
    const EvPlan pl = ev_plan(a);
    IT_CHECK_ARG(a->workspace && it_aligned(a->workspace, 256) && a->workspace_bytes >= pl.total, "%s: a workspace of %zu bytes, 256-byte aligned, is needed", who, pl.total);
    const it_stretch all[] = { { "the workspace", a->workspace, pl.total }, { "weights", a->weights, ((size_t)(G - 1) * (size_t)a->w_head + (size_t)a->n) * 4 },
                               { "kept", a->kept, ((size_t)(G - 1) * (size_t)a->kept_head + (size_t)a->keep) * 4 }, { "k_cache", a->k_cache, it_span(a->n, a->kc_slot, G, a->kc_head, D, 2) },
                               { "v_cache", a->v_cache, it_span(a->n, a->vc_slot, G, a->vc_head, D, 2) } };         // (k and v may lie in one buffer)
    for (int i = 0; i < 3; i++)
        if (const char* x = it_overlaps(all[i], all + i + 1, 4 - i)) return it_fail(IT_EINVAL, "%s: %s overlaps %s", who, all[i].name, x);
    it_ops_device dev;
    if (const int r = it_ops_current(stream, who, &dev)) return r;
    if (const int r = ev_prepare(dev.device)) return r;
    EvParams p;
    char* const ws = (char*)a->workspace;
    p.k = (char*)a->k_cache; p.v = (char*)a->v_cache; p.weights = a->weights; p.status = dev.status_dev;
    p.kept = a->kept ? a->kept : (int*)(ws + pl.kept); p.kept_head = a->kept ? a->kept_head : a->keep;
    p.ranks = (int*)(ws + pl.ranks); p.flags = (unsigned*)(ws + pl.flags);
    p.kc_slot = a->kc_slot * 2; p.kc_head = a->kc_head * 2; p.vc_slot = a->vc_slot * 2; p.vc_head = a->vc_head * 2; p.w_head = a->w_head;
    p.kv_heads = a->kv_heads; p.n = (int)a->n; p.keep = (int)a->keep; p.recent = (int)a->recent; p.row_bytes = a->head_dim * 2;
    p.per = pl.per; p.rank_head = pl.rank_head; p.blocks = pl.blocks; p.nflags = (int)pl.nflags;
    const cudaStream_t st = (cudaStream_t)stream;
    // one CTA a head for short caches, whose passes are all barriers
    if (const int r = pl.cluster == 1 ? ev_select<1>(p, st) : pl.cluster == 8 ? ev_select<8>(p, st) : ev_select<16>(p, st)) return r;
    const unsigned lines = (unsigned)a->kv_heads * ((p.k != nullptr) + (p.v != nullptr));
    if (!lines) return IT_OK;
    IT_CUDA(it_launch_early(k_evict_move, dim3(lines * (unsigned)pl.blocks), dim3(EV_MOVE_THREADS), (size_t)EV_BLOCK * p.row_bytes, st, 1, p));
    return IT_OK;
}
