// The products of tree attention (it_tree_attention.cu) on the 5th-generation tensor cores: tcgen05.mma kind::f16, accumulators in tensor memory.
//
// Both products are formed with the cache as the first operand, whose 128 rows are always full, and the product rows (row t * group + head) as columns, of which there are
// as few as 16:   S^T [128 slots x columns] = K [slots x d] . Q^T,    O^T [d x columns] = V^T [d x slots] . P^T
// so that a decoded token's six rows cost 32 columns and not 128 rows, and everything comes in the layout that it has:
//   K and V tiles   128 slots as boxes of 64 elements of a tensor map, 128-byte swizzle: K is read K-major, V (as V^T) MN-major
//   Q               rows of 128-byte pieces, K-major; f32 activations as two sets of columns, high and low halves, added in f32 when they are read
//   P               [slot][column], MN-major: a thread has one slot (a lane of tensor memory) and stores its columns as 16-byte pieces; high and low halves, two sets of columns
// Softmax warps (two or four groups of four; a group has its share of the columns): scores out of tensor memory, exponentials against a reference that moves only when
// it has to (its maximum over a warp's slots by halving what a lane carries, over the four warps by an ordered atomicMax), P; then the tile before: O^T out of tensor memory into f32 accumulators in registers.  Every tile's product starts from zero and is
// added with a rounded f32 addition: chained over a long run in tensor memory the hardware's truncating accumulation loses f32's last bits (1.3e-5 of the result after 240 tiles of 64
// slots chained in mma.sync accumulators).  Two warps copy, one issues whichever product has its inputs, the next tile's scores or this tile's O.
// What bounds it: 64 columns of f32 activations (128 with the low halves) 2 x 1024 tensor cycles a tile of 128 slots at head dimension 256; few columns: HBM.
#include "it_tree_attention.cuh"
#include "it_route.h"

namespace {

constexpr int TC_SMEM_LIMIT = 227 * 1024, TC_SMALL = 3 * 1024, TC_SLOTS_MAX = 6;
constexpr int TC_JOIN = IT_TREE_JOIN;                            // runs that join in a cluster, at most
constexpr float TC_SHIFT = 6.f, TC_TOP = 15.f;              // p is 2^6 at the reference and may grow to 2^15 before the reference moves

template <bool SPLIT, int NB, int NR> struct TcTree {
    static constexpr int NC = NR * (SPLIT ? 2 : 1);                                           // columns of a tile's scores
    // Columns of P and of O^T: high and low halves whatever the activations.  p rounded once to the cache's type would cost a result over many slots as much as its own last rounding (bf16, one row at
    // 131,071 slots: 0.0022 of the result against 0.0016).  With both, us: 32 over 8 heads of 128, bf16, 12 rows at 8190 slots 19.5 for 18.6, f16, 64 rows 42.9 for 41.7; 24 over 4 of 256, bf16, 64 rows at
    // 30,011 122 for 111; 16 and 32 product rows up to 0.2 more.
    static constexpr int NP = 2 * NR, NCB = NP > 64 ? 2 : 1;                                  // NCB: 64-column blocks of P
    static constexpr int HD = 64 * NB, MT = NB / 2;                                           // M tiles of O^T
    // Accumulators that a score is spread over (f32 activations, where tensor memory has the columns): the hardware truncates at every step, and a chain of 16 of them
    // cost more than half of the result's error at 16 and 32 rows (1.1e-6 of the result after 512 slots).
    static constexpr int PARTS = !SPLIT || NR > 32 ? 1 : NR == 32 ? 2 : NB, SC = PARTS * NC;   // SC: columns of a tile's scores
    // Groups of four softmax warps, and product rows of one.  Four groups for 32 rows and more: a thread's share of a tile is unrolled code that runs a few times, at the speed of
    // instruction-cache misses, and half the rows are half the code.
    static constexpr int WGS = NR >= 32 ? 4 : 2, RW = NR / WGS, SOFT = 128 * WGS, THREADS = SOFT + 128;
    // setmaxnreg deals out the launch's registers: 216 x 256 + 72 x 128 = 168 x 384; 112 x 512 + 32 x 128 = 96 x 640
    static constexpr int REGS = WGS == 2 ? 168 : 96, SOFT_REGS = WGS == 2 ? 216 : 112, OTHER_REGS = WGS == 2 ? 72 : 32;
    static constexpr int QB = NB * NC * 128, PB = NCB * TA_KEYS * 128, BOX = TA_KEYS * 128, SLOT = NB * BOX;
    static constexpr int FIT = (TC_SMEM_LIMIT - TC_SMALL - QB - PB) / SLOT, SLOTS = FIT < TC_SLOTS_MAX ? FIT : TC_SLOTS_MAX;
    static constexpr int KS = (SLOTS + 1) / 2, VS = SLOTS - KS;
    static constexpr int Q = 0, P = QB, KR = P + PB, VR = KR + KS * SLOT, SMALL = VR + VS * SLOT, TOTAL = SMALL + TC_SMALL;
    // offsets from SMALL
    static constexpr int BARS = 0, TMEM = 512, FLAG = 528, MAXES = 576, BASE = 1088, CORR = 1344, FAC = 2112, TROW = 2368;
    static constexpr int TCOLS = 2 * SC + MT * NP, ALLOC = TCOLS <= 64 ? 64 : TCOLS <= 128 ? 128 : TCOLS <= 256 ? 256 : 512;
    static_assert(VS >= 1 && NR % 16 == 0 && NP <= 128 && TCOLS <= 512 && NR <= 64 && NC % 16 == 0 && RW % 8 == 0, "");
    static_assert((2 * KS * NB + 2 * VS * MT + 5 + MT) * 8 <= TMEM, "");
    static_assert(SOFT_REGS * SOFT + OTHER_REGS * 128 <= REGS * THREADS, "");
    static_assert(PB >= TA_MAXROWS * TA_WORDS * 4 + TA_MAXROWS * 4, "the ancestors are worked out in P's place");
    static_assert(KS * SLOT >= NR * TA_KEYS * 4 && KS * SLOT >= NR * HD * 4, "sums and accumulators go through K's place");
};

// Shared-memory descriptors, 128-byte swizzle, version 1.  K-major: 8-row groups 1024 bytes apart.  MN-major: blocks of 64 elements `block` bytes apart, groups of 8 along K 1024 bytes apart.
__device__ __forceinline__ unsigned long long desc_k(unsigned addr) {
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned long long desc_mn(unsigned addr, unsigned block) {
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(block >> 4) << 16) | ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 instruction descriptor: D f32, A and B f16 or bf16, M 128, N columns; bits 15 and 16: A and B MN-major
template <class T> __host__ __device__ constexpr unsigned idesc(int n, bool mn) {
    constexpr unsigned ty = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (ty << 7) | (ty << 10) | (mn ? (1u << 15) | (1u << 16) : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(unsigned d, unsigned long long a, unsigned long long b, unsigned id, bool acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}"
                 :: "r"(d), "l"(a), "l"(b), "r"(id), "r"(acc ? 1u : 0u), "r"(0u) : "memory");
}
// The bounded waits of it_pipe.cuh with their retries rolled up: the kernel has a dozen of them, and what matters here is how much code lies between its parts.
__device__ __forceinline__ bool tc_wait(unsigned bar, unsigned parity, volatile int* abort_flag, int* status, int site) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
#pragma unroll 1
    while (!mbar_test_hint(bar, parity, IT_MBAR_SLEEP_NS)) {
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_CLOCKS) { if (!*abort_flag) atomicExch(status, site); *abort_flag = 1; return false; }
    }
    return true;
}
// For a warp that goes on as one: true in every lane or in none.
__device__ __forceinline__ bool tc_wait_warp(unsigned bar, unsigned parity, volatile int* abort_flag, int* status, int site) {
    return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag, status, site));
}
__device__ __forceinline__ void commit_to(unsigned bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ bool elect_one() {
    unsigned e;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// Neighbouring columns of this thread's lane.
__device__ __forceinline__ void tm_ld(float (&v)[8], unsigned a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_ld(float (&v)[16], unsigned a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_ld(float (&v)[32], unsigned a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                   "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]) : "r"(a) : "memory");
}
// Waits for the loads; the values pass through it so that nothing that uses them moves in front.
template <int N> __device__ __forceinline__ void tm_wait(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+f"(v[i]));
}
// Maximum over the warp of each of N values (NaN left out, as by fmaxf): lane r gets that of value r, for r < N.  Halves what a lane carries at every step; a redux a value costs the
// sub-core 16 cycles each, 1050 for four warps of 16 values.
template <int N> __device__ __forceinline__ float warp_max(float (&v)[N], int lane) {
#pragma unroll
    for (int h = N / 2; h > 0; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; i++) {
            const float keep = up ? v[i + h] : v[i], give = up ? v[i] : v[i + h];
            v[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, h));
        }
    }
#pragma unroll
    for (int h = N; h < 32; h <<= 1) v[0] = fmaxf(v[0], __shfl_xor_sync(0xffffffffu, v[0], h));
    return v[0];
}
// Integers in the order of the floats.
__device__ __forceinline__ int ordered(float v) { const int i = __float_as_int(v); return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
template <int N> __device__ __forceinline__ void warp_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void warp_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }
// Barriers of one group of four warps, and of all WGS groups.  The numbers are constants: a barrier whose number is a register makes the compiler reserve all sixteen.
__device__ __forceinline__ void group_sync(int wg) {
    if (wg == 0) asm volatile("bar.sync 1, 128;" ::: "memory"); else if (wg == 1) asm volatile("bar.sync 2, 128;" ::: "memory");
    else if (wg == 2) asm volatile("bar.sync 3, 128;" ::: "memory"); else asm volatile("bar.sync 4, 128;" ::: "memory");
}
template <int WGS> __device__ __forceinline__ void groups_sync() { asm volatile("bar.sync 5, %0;" :: "n"(128 * WGS) : "memory"); }
// Whether any thread of a group says so, with a barrier of the group.
template <int N> __device__ __forceinline__ unsigned group_or(unsigned q) {
    unsigned r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 q, %1, 0;\nbarrier.cta.red.or.pred p, %2, 128, q;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r) : "r"(q), "n"(N) : "memory");
    return r;
}
__device__ __forceinline__ bool group_any(int wg, bool q) { return (wg == 0 ? group_or<1>(q) : wg == 1 ? group_or<2>(q) : wg == 2 ? group_or<3>(q) : group_or<4>(q)) != 0; }

// The cluster's barrier, and its CTAs' shared memory.
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ unsigned cluster_addr(unsigned a, int rank) { unsigned r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank)); return r; }
__device__ __forceinline__ float2 ld_cluster2(unsigned a, int rank) {
    float2 v; asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(a, rank)) : "memory"); return v;
}
__device__ __forceinline__ float4 ld_cluster4(unsigned a, int rank) {
    float4 v; asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(a, rank)) : "memory"); return v;
}

// Product rows [r0, r0 + NR) of KV head g as columns of Q^T; for each the factor from the product to log2 of its exponential, and its row t (rows behind the last: the
// last one's).  A warp has all of its rows' loads under way at once: one after the other they were 7 us of a 64-row tile.
template <class T, bool SPLIT, int NB, int NR, int NW>
__device__ void tc_load_q(const TaParams& p, unsigned char* q, float* fac, int* trow, int g, int r0, int warp, int lane) {
    using L = TcTree<SPLIT, NB, NR>;
    constexpr int N = (NR + NW - 1) / NW;
    TaRow<T, SPLIT> x[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int i = warp + k * NW, r = r0 + i, t = min(ta_row(p, r), p.rows - 1), h = g * p.group + r - t * p.group;
        if (i < NR && lane == 0) trow[i] = t;
        x[k].load(p, i < NR && r < p.prows && 8 * lane < p.dim, t, h, lane);
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int i = warp + k * NW;
        if (i >= NR) break;
        unsigned hi[4], lo[4];
        const float f = x[k].halves(p, hi, lo);
        if (lane < NB * 8) {
            const unsigned at = (unsigned)((lane >> 3) * L::NC * 128) + swz(i, lane & 7);
            *reinterpret_cast<uint4*>(q + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) *reinterpret_cast<uint4*>(q + at + NR * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (lane == 0) fac[i] = f;
    }
}

// Whether row t sees tree slot i, by walking up; for the rare case only.
__device__ __noinline__ bool tc_walk(const int* parents, int t, int i) {
    if (i > t) return false;
    if (!parents) return true;
    while (t > i) { const int q = parents[t]; if (q < 0 || q >= t) return false; t = q; }
    return t == i;
}

template <class T, bool SPLIT, int NB, int NR>
__global__ void __launch_bounds__(TcTree<SPLIT, NB, NR>::THREADS, 1)
k_tree_attention_tc(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TaParams p) {
    using L = TcTree<SPLIT, NB, NR>;
    using TA = typename std::conditional<SPLIT, float, T>::type;
    constexpr int NC = L::NC, NP = L::NP, RW = L::RW, HD = L::HD, KS = L::KS, VS = L::VS, WGS = L::WGS, MT = L::MT, W0 = 4 * WGS;       // W0: the first warp behind the softmax warps
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, g = blockIdx.y, r0 = blockIdx.z * NR;
    unsigned char* const small = smem + L::SMALL;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(small + L::FLAG);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(small + L::TMEM);
    int* maxes = reinterpret_cast<int*>(small + L::MAXES);              // [2][NR]
    float* base_s = reinterpret_cast<float*>(small + L::BASE);          // [NR]
    float* corr_s = reinterpret_cast<float*>(small + L::CORR);          // [2][NR]: a group's rows are its own, the tile before is taken over after this one's scores
    float* fac = reinterpret_cast<float*>(small + L::FAC);              // [NR]
    int* trow = reinterpret_cast<int*>(small + L::TROW);                // [NR]
    const unsigned bars = smem_u32(small + L::BARS);
    // K in boxes of 64 elements, V in pairs of them (an M tile of O^T): each has barriers of its own, so that the next tile's first box is asked for when this tile's is read
    const unsigned kfull = bars, kempty = kfull + 8 * KS * NB, vfull = kempty + 8 * KS * NB, vempty = vfull + 8 * VS * MT, sfull = vempty + 8 * VS * MT, sfree = sfull + 16, pfull = sfree + 16, ofull = pfull + 8;       // (one an M tile)
    const unsigned kring = smem_u32(smem + L::KR), vring = smem_u32(smem + L::VR);

    if (warp == W0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" :: "l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&vmap) : "memory");
        *abort_flag = (smem_u32(smem) & 1023u) != 0;                 // the swizzle counts on it; never seen
#pragma unroll 1
        for (int s = 0; s < 2 * (KS * NB + VS * MT); s++) mbar_init(bars + 8 * s, 1);
        for (int s = 0; s < 2; s++) { mbar_init(sfull + 8 * s, 1); mbar_init(sfree + 8 * s, W0); }
        mbar_init(pfull, W0);
        for (int m = 0; m < MT; m++) mbar_init(ofull + 8 * m, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W0 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)), "r"((unsigned)L::ALLOC) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid < 2 * NR) maxes[tid] = ordered(-INFINITY);
    __syncwarp();
    // The kernel may have begun while the one before it still ran; from here on it reads what that one wrote.  Only then may the kernels behind it begin: they read the caller's
    // gate, cache and parents before they wait for this one.
    asm volatile("griddepcontrol.wait;\ngriddepcontrol.launch_dependents;" ::: "memory");
    const int cached = ta_cached(p), total = cached + p.rows, tiles = (total + TA_KEYS - 1) / TA_KEYS;
    // this run's tiles: the first `tiles % splits` runs have one more
    const int per = (int)((unsigned)tiles / (unsigned)p.splits), more = tiles - per * p.splits, tile0 = split * per + min(split, more), n = per + (split < more ? 1 : 0);
    // Box b of tile i of K, pair m of tile i of V, when their places are free; copies of K and V have a warp each, since they wait for different products.
    auto load_k = [&](int i, int b) {
        const unsigned at = (unsigned)(i % KS * NB + b);
        mbar_expect_tx(kfull + 8 * at, L::BOX);
        tma_load_3d(kring + at * L::BOX, &kmap, 64 * b, (tile0 + i) * TA_KEYS, g, kfull + 8 * at);
    };
    auto load_v = [&](int i, int m) {
        const unsigned at = (unsigned)(i % VS * MT + m);
        mbar_expect_tx(vfull + 8 * at, 2 * L::BOX);
        tma_load_3d(vring + 2 * at * L::BOX, &vmap, 128 * m, (tile0 + i) * TA_KEYS, g, vfull + 8 * at);
        tma_load_3d(vring + (2 * at + 1) * L::BOX, &vmap, 128 * m + 64, (tile0 + i) * TA_KEYS, g, vfull + 8 * at);
    };
    if (warp == W0 && lane == 0 && n > 0) {                          // the first tile before anything else
#pragma unroll 1
        for (int b = 0; b < NB; b++) load_k(0, b);
#pragma unroll 1
        for (int m = 0; m < MT; m++) load_v(0, m);
    }
    __syncwarp();
    tc_load_q<T, SPLIT, NB, NR, L::THREADS / 32>(p, smem + L::Q, fac, trow, g, r0, warp, lane);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // Q before the products read it
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = *tmem_slot, otm = tmem + 2 * L::SC;

    float2* const ml = reinterpret_cast<float2*>(smem + L::P);       // [NR], at the end: references and sums of the rows
    float* const os = reinterpret_cast<float*>(smem + L::KR);        // [NR][HD], at the end: accumulators
    if (warp < W0) {
        warp_regs_inc<L::SOFT_REGS>();
        const int wg = warp >> 2, quad = warp & 3, key = quad * 32 + lane;
        const unsigned lanes = (unsigned)(quad * 32) << 16;
        const unsigned oaddr = otm + lanes + wg * RW;               // the accumulators: elements `key` and 128 + `key` of the head, the group's product rows
        float acc[MT][RW], l[RW], mrun = -INFINITY;                 // mrun: the reference of row `lane` of the group
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int r = 0; r < RW; r++) acc[m][r] = 0.f;
#pragma unroll
        for (int r = 0; r < RW; r++) l[r] = 0.f;
        bool ok = true;
        // Which of the group's product rows see this thread's slot, for the tiles that reach behind the cached slots; while the first scores are formed.
        const int first_masked = cached / TA_KEYS - tile0;
        unsigned vis[3] = { 0, 0, 0 };
        if (n > first_masked && n > 0) {
            unsigned (*anc)[TA_WORDS] = reinterpret_cast<unsigned (*)[TA_WORDS]>(smem + L::P);
            if (p.parents) ta_ancestors<L::SOFT>(anc, reinterpret_cast<int*>(smem + L::P + TA_MAXROWS * TA_WORDS * 4), p.parents, p.rows, tid, [] { groups_sync<WGS>(); });
#pragma unroll
            for (int k = 0; k < 3; k++) {
                if (first_masked + k >= n) break;
                const int i = (tile0 + first_masked + k) * TA_KEYS + key - cached;           // the slot among the rows' own
                unsigned m = i < 0 ? 0xffffffffu : 0u;
                if (i >= 0 && i < p.rows) {
#pragma unroll 4
                    for (int r = 0; r < RW; r++) {
                        const int t = trow[wg * RW + r];
                        if (p.parents ? (anc[t][i >> 5] >> (i & 31)) & 1u : i <= t) m |= 1u << r;
                    }
                }
                vis[k] = m;
            }
            groups_sync<WGS>();                                     // before P takes the place of the ancestors
        }
        int exact = 0;                                              // references moved so far
        // O^T of tile i.  What the first M tile gave is taken over while the second is still under way.
        auto collect = [&](int i) {
            const float* const c = corr_s + (i & 1) * NR + wg * RW;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                ok = ok && tc_wait_warp(ofull + 8 * m, (unsigned)i & 1u, abort_flag, p.status, 52);
                fence_after();
                constexpr int CH = RW < 16 ? RW : 16;
#pragma unroll
                for (int k = 0; k < RW; k += CH) {
                    float u[CH], v[CH];
                    tm_ld(u, oaddr + m * NP + k);
                    tm_ld(v, oaddr + m * NP + NR + k);
                    tm_wait(u);
#pragma unroll
                    for (int e = 0; e < CH; e++) { asm volatile("" : "+f"(v[e])); u[e] += v[e]; }
#pragma unroll
                    for (int e = 0; e < CH; e++) acc[m][k + e] = fmaf(acc[m][k + e], c[k + e], u[e]);
                }
            }
            fence_before();
        };
#pragma unroll 1
        for (int i = 0; i <= n; i++) {                              // softmax of tile i, O^T of tile i - 1, P of tile i
            unsigned hi[RW / 2], lo[RW / 2];
            const bool masked = i >= first_masked;
            if (i < n) {
                const int buf = i & 1;
                ok = ok && tc_wait_warp(sfull + 8 * buf, (unsigned)(i >> 1) & 1u, abort_flag, p.status, 51);
                fence_after();
                float x[RW];
                const unsigned sa = tmem + lanes + buf * L::SC + wg * RW;
                if constexpr (SPLIT) {                              // the parts' low halves, then their high halves
                    float y[2 * L::PARTS][RW];
#pragma unroll
                    for (int k = 0; k < 2 * L::PARTS; k++) tm_ld(y[k], sa + (k % L::PARTS) * NC + (k < L::PARTS ? NR : 0));
                    tm_wait(y[0]);
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        x[r] = y[0][r];
#pragma unroll
                        for (int k = 1; k < 2 * L::PARTS; k++) { asm volatile("" : "+f"(y[k][r])); x[r] += y[k][r]; }
                    }
                } else { tm_ld(x, sa); tm_wait(x); }
                fence_before();
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(sfree + 8 * buf);
                // Exponents against the rows' references.  A reference need not be the maximum: it moves when an exponent would pass f16's range, in the first tile, and in
                // masked tiles (a row may have seen nothing before), which spares all other tiles the maximum over slots.
                const float *const f = fac + wg * RW, *const bs = base_s + wg * RW;
                float* const c = corr_s + (i & 1) * NR + wg * RW;
                bool move = i == 0 || masked;
                const unsigned see = masked ? (i == first_masked ? vis[0] : i == first_masked + 1 ? vis[1] : vis[2]) : 0xffffffffu;
                if (p.scores) {                                     // for the received weights
                    float* const s = p.scores + ((long long)g * p.prows + r0 + wg * RW) * p.s_row + (tile0 + i) * TA_KEYS + key;
#pragma unroll
                    for (int r = 0; r < RW; r++)
                        if (r0 + wg * RW + r < p.prows) __stcg(s + r * p.s_row, (see >> r) & 1u ? x[r] * f[r] : -INFINITY);
                }
                float y[RW];
                if (!move) {
                    float top = -INFINITY;
#pragma unroll
                    for (int r = 0; r < RW; r++) { y[r] = fmaf(x[r], f[r], -bs[r]); top = fmaxf(top, y[r]); }
                    move = group_any(wg, top > TC_TOP);             // the same answer in all four warps
                }
                if (move) {
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        x[r] = (see >> r) & 1u ? x[r] * f[r] : -INFINITY;
                        y[r] = x[r];
                    }
                    const float mine = warp_max(y, lane);
                    int* const best = maxes + (exact & 1) * NR + wg * RW;
                    exact++;
                    if (lane < RW) atomicMax(best + lane, ordered(fmaxf(mrun, mine)));
                    group_sync(wg);
                    if (lane < RW) {                                // the four warps write the same values
                        const float m = unordered(best[lane]), ref = m == -INFINITY ? 0.f : m;
                        c[lane] = ex2(mrun - ref);
                        base_s[wg * RW + lane] = ref - TC_SHIFT;
                        mrun = m;
                    }
                    __syncwarp();
#pragma unroll
                    for (int r = 0; r < RW; r++) { y[r] = x[r] - bs[r]; l[r] *= c[r]; }
                } else if (lane < RW) c[lane] = 1.f;
#pragma unroll
                for (int r = 0; r < RW; r += 2) {
                    const float a = ex2(y[r]), b = ex2(y[r + 1]);
                    l[r] += a; l[r + 1] += b;
                    hi[r / 2] = Ta16<T>::pack(a, b);
                    const float2 h = Ta16<T>::unpack(hi[r / 2]);
                    lo[r / 2] = Ta16<T>::pack(a - h.x, b - h.y);
                }
            }
            if (i > 0) collect(i - 1);                               // frees O^T and P
            if (i == n) break;
            unsigned char* const prow = smem + L::P + key * 128;
#pragma unroll
            for (int k = 0; k < RW / 8; k++) {
                const int ch = wg * (RW / 8) + k, cl = ch + NR / 8;       // 16-byte pieces of the high and the low columns
                *reinterpret_cast<uint4*>(prow + ((ch ^ (key & 7)) << 4)) = make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
                *reinterpret_cast<uint4*>(prow + (cl >> 3) * L::BOX + (((cl & 7) ^ (key & 7)) << 4)) = make_uint4(lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
            }
            if (masked) {
                // V elements that are not finite leave the product and go to the rows that see their slot; in front of this tile's correction, which therefore must not be 0 (0 * inf)
                float* const c = corr_s + (i & 1) * NR + wg * RW;
#pragma unroll
                for (int r = 0; r < RW; r++)
                    if (c[r] == 0.f) {
#pragma unroll
                        for (int m = 0; m < MT; m++) acc[m][r] = 0.f;
                    }
                const int j0 = (tile0 + i) * TA_KEYS, from = max(cached - j0, 0), to = min(TA_KEYS, p.cached + p.rows - j0);
                bool any[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    ok = ok && tc_wait_warp(vfull + 8 * (i % VS * MT + m), (unsigned)(i / VS) & 1u, abort_flag, p.status, 54);
                    const unsigned char* const v = smem + L::VR + (i % VS) * L::SLOT + (2 * m + (key >> 6)) * L::BOX + (key & 7) * 2;
                    any[m] = false;
#pragma unroll 1
                    for (int k = from; k < to; k++) {
                        const unsigned short raw = *reinterpret_cast<const unsigned short*>(v + k * 128 + ((((key & 63) >> 3) ^ (k & 7)) << 4));
                        if ((raw & Ta16<T>::EXP) != Ta16<T>::EXP) continue;
                        any[m] = true;
                        unsigned rows = 0;
#pragma unroll 1
                        for (int r = 0; r < RW; r++)
                            if (j0 + k - cached < p.rows && tc_walk(p.parents, trow[wg * RW + r], j0 + k - cached)) rows |= 1u << r;
                        const float bad = Ta16<T>::unpack(raw).x;
#pragma unroll
                        for (int r = 0; r < RW; r++) if ((rows >> r) & 1u) acc[m][r] += bad;
                    }
                }
                groups_sync<WGS>();                         // all groups have looked at the elements that one of them clears, and at the corrections
                if (lane < RW && c[lane] == 0.f) c[lane] = 1.f;          // (the four warps write the same)
#pragma unroll
                for (int m = 0; m < MT; m++)
                    if (any[m] && wg == 0) {
                        unsigned char* const v = smem + L::VR + (i % VS) * L::SLOT + (2 * m + (key >> 6)) * L::BOX + (key & 7) * 2;
#pragma unroll 1
                        for (int k = from; k < to; k++) {
                            unsigned short* e = reinterpret_cast<unsigned short*>(v + k * 128 + ((((key & 63) >> 3) ^ (k & 7)) << 4));
                            if ((*e & Ta16<T>::EXP) == Ta16<T>::EXP) *e = 0;
                        }
                    }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(pfull);
        }
        // ---- every product is done: the rings are free.  The rows' sums are those of the slots' threads.
        float* const sums = reinterpret_cast<float*>(smem + L::KR);            // [NR][128]
#pragma unroll
        for (int r = 0; r < RW; r++) sums[(wg * RW + r) * TA_KEYS + key] = l[r];
        group_sync(wg);
        const bool bad = *abort_flag != 0;
#pragma unroll
        for (int r = 0; r < RW / 4; r++) {
            const int row = wg * RW + quad + 4 * r;
            const float4 e = *reinterpret_cast<const float4*>(sums + row * TA_KEYS + 4 * lane);
            float v = (e.x + e.y) + (e.z + e.w);
#pragma unroll
            for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
            if (lane == 0) ml[row].y = bad ? NAN : v;
        }
        if (quad == 0 && lane < RW) ml[wg * RW + lane].x = mrun == -INFINITY ? mrun : base_s[wg * RW + lane];
        if (!p.joined) {
            const size_t at = ((size_t)split * p.kv_heads + g) * p.pad_rows + r0;
            float* const o = p.part_o + (at + wg * RW) * HD + key;
#pragma unroll
            for (int r = 0; r < RW; r++)
                if (r0 + wg * RW + r < p.prows) {
#pragma unroll
                    for (int m = 0; m < MT; m++) __stcg(o + r * HD + 128 * m, acc[m][r]);
                }
            groups_sync<WGS>();
            if (tid < NR) p.part_ml[at + tid] = ml[tid];
        } else {
            groups_sync<WGS>();                                     // the sums, in whose place the accumulators go, are read
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int r = 0; r < RW; r++) os[(wg * RW + r) * HD + 128 * m + key] = acc[m][r];
            // The runs of a short cache are a cluster, and join here: a run finishes every splits-th row, four elements a thread, reading the others' sums and accumulators
            // from their shared memory.  Saves the partial results and a launch.
            cluster_sync();
            constexpr int LN = HD / 4, STEP = L::SOFT / LN;          // threads of a row, rows at once
            const int c = tid % LN * 4;
            const unsigned mla = smem_u32(ml), osa = smem_u32(os) + 4 * c;
#pragma unroll 1
            for (int q = tid / LN; c < p.dim; q += STEP) {
                const int r = split + p.splits * q, row = r0 + r;
                if (r >= NR || row >= p.prows) break;
                const int t = trow[r], h = g * p.group + row - t * p.group;
                float z[4] = { 0.f, 0.f, 0.f, 0.f };
                if (p.gate) load4((const TA*)p.gate + t * p.g_row + h * p.g_head + c, z);
                float2 e[TC_JOIN];
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < TC_JOIN; k++) {
                    e[k] = k < p.splits ? ld_cluster2(mla + 8 * r, k) : make_float2(-INFINITY, 0.f);
                    top = fmaxf(top, e[k].x);
                }
                const float ref = top == -INFINITY ? 0.f : top;
                float sum = 0.f, o[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                for (int k = 0; k < TC_JOIN; k++) {
                    if (k >= p.splits || (e[k].x == -INFINITY && e[k].y == 0.f)) continue;       // saw nothing
                    const float w = ex2(e[k].x - ref);
                    const float4 v = ld_cluster4(osa + (unsigned)(r * HD * 4), k);
                    sum = fmaf(e[k].y, w, sum);
                    o[0] = fmaf(v.x, w, o[0]); o[1] = fmaf(v.y, w, o[1]); o[2] = fmaf(v.z, w, o[2]); o[3] = fmaf(v.w, w, o[3]);
                }
                if (p.stats && c == 0) p.stats[(size_t)g * p.pad_rows + row] = make_float2(ref, sum);
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] *= inv;
                if (p.gate) {
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] /= 1.f + __expf(-z[i]);
                }
                store4((TA*)p.out + t * p.o_row + h * p.o_head + c, o);
            }
            __syncwarp();
            cluster_sync();                                         // nobody leaves while its shared memory may still be read
        }
    } else {
        warp_regs_dec<L::OTHER_REGS>();
        // Leaving after a wait that ran out: only when every copy has landed (bounded).
        auto landed = [&](unsigned full, int from, int to, int ring) {
#pragma unroll 1
            for (int k = max(from, to - ring); k < to; k++) { const long long t0 = clock64(); while (!mbar_test(full + 8 * (k % ring), (unsigned)(k / ring) & 1u) && clock64() - t0 < WAIT_CLOCKS) { } }
        };
        if (warp == W0) {
            // ---------------- copies of K
            if (lane == 0) {
                int k = NB;                         // boxes asked for
#pragma unroll 1
                for (; k < n * NB; k++) {
                    if (k >= KS * NB && !tc_wait(kempty + 8 * (k % (KS * NB)), ((unsigned)(k / (KS * NB)) & 1u) ^ 1u, abort_flag, p.status, 55)) break;
                    load_k(k / NB, k % NB);
                }
                if (*abort_flag && n > 0) landed(kfull, 0, k, KS * NB);
            }
        } else if (warp == W0 + 2) {
            // ---------------- copies of V
            if (lane == 0) {
                int k = MT;
#pragma unroll 1
                for (; k < n * MT; k++) {
                    if (k >= VS * MT && !tc_wait(vempty + 8 * (k % (VS * MT)), ((unsigned)(k / (VS * MT)) & 1u) ^ 1u, abort_flag, p.status, 56)) break;
                    load_v(k / MT, k % MT);
                }
                if (*abort_flag && n > 0) landed(vfull, 0, k, VS * MT);
            }
        } else if (warp == W0 + 1) {
            // ---------------- products: the scores of tile si, O^T of tile oi, whichever has its inputs.  Loops, not straight code: see WGS.
            if (elect_one()) {
                const unsigned long long qd = desc_k(smem_u32(smem + L::Q)), pd = desc_mn(smem_u32(smem + L::P), L::BOX);
                int si = 0, kb = 0, oi = 0, om = 0; long long since = clock64();          // tile of the scores, box of K, tile and M tile of the products that come next
#pragma unroll 1
                while (oi < n) {
                    const unsigned va = (unsigned)(oi % VS * MT + om), ka = (unsigned)(kb % (KS * NB));
                    if (oi < si && (om > 0 || mbar_poll(pfull, (unsigned)oi & 1u)) && mbar_poll(vfull + 8 * va, (unsigned)(oi / VS) & 1u)) {
                        fence_after();
                        unsigned long long vd = desc_mn(vring + 2 * va * L::BOX, L::BOX), pb = pd;
#pragma unroll 1
                        for (int k = 0; k < TA_KEYS / 16; k += 4) {
#pragma unroll
                            for (int j = 0; j < 4; j++) mma_f16(otm + om * NP, vd + (unsigned)(j * 2048 >> 4), pb + (unsigned)(j * 2048 >> 4), idesc<T>(NP, true), k + j > 0);          // 16 slots a step
                            vd += (unsigned)(4 * 2048 >> 4); pb += (unsigned)(4 * 2048 >> 4);
                        }
                        commit_to(ofull + 8 * om); commit_to(vempty + 8 * va);
                        if (++om == MT) { om = 0; oi++; }
                        since = clock64();
                    } else if (si < n && (kb % NB || mbar_poll(sfree + 8 * (si & 1), ((unsigned)(si >> 1) & 1u) ^ 1u)) && mbar_poll(kfull + 8 * ka, (unsigned)(si / KS) & 1u)) {
                        // a box at a time, so that a product whose P comes meanwhile does not wait for K
                        const int b = kb % NB;
                        fence_after();
                        const unsigned long long kd = desc_k(kring + ka * L::BOX), qb = qd + (unsigned)(b * NC * 128 >> 4);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_f16(tmem + (si & 1) * L::SC + b * L::PARTS / NB * NC, kd + (unsigned)(k * 32 >> 4), qb + (unsigned)(k * 32 >> 4), idesc<T>(NC, false), b % (NB / L::PARTS) + k > 0);     // 16 elements of the head a step
                        commit_to(kempty + 8 * ka);
                        if (b == NB - 1) { commit_to(sfull + 8 * (si & 1)); si++; }
                        kb++; since = clock64();
                    } else if (*abort_flag) break;
                    else if (clock64() - since > WAIT_CLOCKS) { if (!*abort_flag) atomicExch(p.status, 59); *abort_flag = 1; break; }
                }
                // the last commits must find the CTA's shared memory still its own (bounded)
                landed(kempty, 0, kb, KS * NB); landed(vempty, 0, oi * MT + om, VS * MT);
            }
        }
        __syncwarp();
        if (p.joined) { cluster_sync(); cluster_sync(); }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == W0 + 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((unsigned)L::ALLOC) : "memory");
    }
}

// ---- received weight, where the scores are not kept -----------------------------------------------------------------------------
// The scores of a 128-slot tile once more, against the finished reference and sum of every product row: a thread has a slot and adds up its columns, so that nothing crosses
// threads but the two groups' halves.  A CTA walks tiles of a KV head; product rows are brought in NR at a time for every tile.  The next scores are
// formed while the last ones' exponentials are, and the next tile of K is on its way (one tile a CTA: 21 us at 8192 slots and 9 rows, most of it start-up).
constexpr int TW_THREADS = 256, TW_ROWS = 64;
template <bool SPLIT, int NB, int NR> struct TcWeights {
    using A = TcTree<SPLIT, NB, NR>;
    static constexpr int Q = 0, K = A::QB, ANC = K + 2 * A::SLOT, JUMP = ANC + TA_MAXROWS * TA_WORDS * 4, ROW = JUMP + TA_MAXROWS * 4, HALF = ROW + 3 * 4 * NR * 4, BARS = HALF + 2 * TA_KEYS * 4, TMEM = BARS + 32,
                         FLAG = TMEM + 16, TOTAL = FLAG + 16;
    static constexpr int ALLOC = 2 * A::NC < 32 ? 32 : 2 * A::NC;
    static_assert(TOTAL <= TC_SMEM_LIMIT, "");
};
template <class T, bool SPLIT, int NB, int NR>
__global__ void __launch_bounds__(TW_THREADS)
k_tree_weights_tc(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ TaParams p) {
    using L = TcTree<SPLIT, NB, NR>;
    using W = TcWeights<SPLIT, NB, NR>;
    constexpr int NC = L::NC, RW = NR / 2;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = blockIdx.y;
    const int wg = warp >> 2, quad = warp & 3, key = quad * 32 + lane;
    const int cached = ta_cached(p), total = cached + p.rows, tiles = (total + TA_KEYS - 1) / TA_KEYS;
    const int nt = ((int)blockIdx.x < tiles) ? (tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;      // tiles blockIdx.x, + gridDim.x, ...
    if (nt == 0) { asm volatile("griddepcontrol.wait;" ::: "memory"); return; }
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + W::FLAG);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + W::TMEM);
    const unsigned kfull = smem_u32(smem + W::BARS), sfull = kfull + 16;
    unsigned (*anc)[TA_WORDS] = reinterpret_cast<unsigned (*)[TA_WORDS]>(smem + W::ANC);
    float* const row = reinterpret_cast<float*>(smem + W::ROW);       // [3][factor, base, 1 / sum, row t][NR]: a slow warp may still read step q - 1 while a fast one brings q + 1
    auto load = [&](int j) {
        const unsigned bar = kfull + 8 * (j & 1);
        mbar_expect_tx(bar, L::SLOT);
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_3d(smem_u32(smem + W::K) + (j & 1) * L::SLOT + b * L::BOX, &kmap, 64 * b, ((int)blockIdx.x + j * (int)gridDim.x) * TA_KEYS, g, bar);
    };
    if (tid == 0) {
        *abort_flag = 0;
        for (int k = 0; k < 4; k++) mbar_init(kfull + 8 * k, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        load(0);
        if (nt > 1) load(1);
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)), "r"((unsigned)W::ALLOC) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int last_tile = (int)blockIdx.x + (nt - 1) * (int)gridDim.x;
    if (p.parents && (last_tile + 1) * TA_KEYS > cached) ta_ancestors<TW_THREADS>(anc, reinterpret_cast<int*>(smem + W::JUMP), p.parents, p.rows, tid, [] { __syncthreads(); });
    asm volatile("griddepcontrol.wait;" ::: "memory");                // the statistics come from the kernel before
    const int steps = (p.prows + NR - 1) / NR;
    auto bring = [&](int i, int q) {                                  // product rows of step i, and their statistics
        float* const rw = row + (q % 3) * 4 * NR;
        tc_load_q<T, SPLIT, NB, NR, TW_THREADS / 32>(p, smem + W::Q, rw, reinterpret_cast<int*>(rw + 3 * NR), g, i * NR, warp, lane);
        if (tid < NR) {
            const int r = i * NR + tid;
            const float2 st = r < p.prows ? __ldcg(&p.stats[(size_t)g * p.pad_rows + r]) : make_float2(0.f, 0.f);
            rw[NR + tid] = st.x; rw[2 * NR + tid] = st.y == 0.f ? 0.f : 1.f / st.y;          // rows behind the last: nothing
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    bring(0, 0);
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = *tmem_slot;
    const unsigned long long qd = desc_k(smem_u32(smem + W::Q));
    bool ok = true;
    auto issue = [&](int j, int q) {                                  // the scores of step q, a step of tile j
        if (warp == 0) {
            ok = ok && tc_wait_warp(kfull + 8 * (j & 1), (unsigned)(j >> 1) & 1u, abort_flag, p.status, 61);
            if (elect_one()) {
                const unsigned long long kd = desc_k(smem_u32(smem + W::K) + (j & 1) * L::SLOT);
                fence_after();
#pragma unroll 1
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_f16(tmem + (q & 1) * NC, kd + (unsigned)((b * L::BOX + k * 32) >> 4), qd + (unsigned)((b * NC * 128 + k * 32) >> 4), idesc<T>(NC, false), b + k > 0);
                commit_to(sfull + 8 * (q & 1));
            }
            __syncwarp();
        }
    };
    issue(0, 0);
    int q = 0;
#pragma unroll 1
    for (int j = 0; j < nt; j++) {
        const int tile = (int)blockIdx.x + j * (int)gridDim.x;
        const bool masked = (tile + 1) * TA_KEYS > cached;
        float sum = 0.f;
#pragma unroll 1
        for (int i = 0; i < steps; i++, q++) {
            ok = ok && tc_wait_warp(sfull + 8 * (q & 1), (unsigned)(q >> 1) & 1u, abort_flag, p.status, 62);
            fence_after();
            const bool last = i + 1 == steps;
            if (last && tid == 0 && j + 2 < nt && ok) load(j + 2);    // every product with this tile is done
            if (!last || j + 1 < nt) {
                bring(last ? 0 : i + 1, q + 1);                       // the products of step q are done with Q
                fence_before();
                __syncthreads();                                      // everyone has read the scores of step q - 1
                issue(last ? j + 1 : j, q + 1);
            }
            float x[RW];
            const unsigned sa = tmem + ((unsigned)(quad * 32) << 16) + (q & 1) * NC + wg * RW;
            tm_ld(x, sa);
            if constexpr (SPLIT) {
                float y[RW];
                tm_ld(y, sa + NR);
                tm_wait(x);
#pragma unroll
                for (int r = 0; r < RW; r++) { asm volatile("" : "+f"(y[r])); x[r] += y[r]; }
            } else tm_wait(x);
            fence_before();
            const float* const rw = row + q % 3 * 4 * NR + wg * RW;
            if (!masked) {
#pragma unroll
                for (int r = 0; r < RW; r++) {                        // rows behind the last are zeros: 0 * inf of a key is NaN, and does not count
                    const float inv = rw[2 * NR + r];
                    sum = inv == 0.f ? sum : fmaf(ex2(fmaf(x[r], rw[r], -rw[NR + r])), inv, sum);
                }
            } else {
                // a masked score does not count, whatever it is, nor does a row behind the last
                const int t0 = tile * TA_KEYS + key;
#pragma unroll
                for (int r = 0; r < RW; r++) {
                    const float inv = rw[2 * NR + r], e = ex2(fmaf(x[r], rw[r], -rw[NR + r])) * inv;
                    if (inv != 0.f && ta_sees(p, anc, reinterpret_cast<const int*>(rw)[3 * NR + r], t0, cached)) sum += e;
                }
            }
        }
        float* const half = reinterpret_cast<float*>(smem + W::HALF) + (j & 1) * TA_KEYS;
        if (wg == 1) half[key] = sum;
        __syncthreads();
        if (wg == 0 && tile * TA_KEYS + key < total) {
            float* w = p.weights + (long long)g * p.w_head + tile * TA_KEYS + key;
            *w = ok && !*abort_flag ? *w + (sum + half[key]) : NAN;
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        if (*abort_flag && lane == 0)                                 // leave only after the copies have landed (bounded)
            for (int j = nt > 2 ? nt - 2 : 0; j < nt; j++) { const long long t0 = clock64(); while (!mbar_test(kfull + 8 * (j & 1), (unsigned)(j >> 1) & 1u) && clock64() - t0 < WAIT_CLOCKS) { } }
        __syncwarp();
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((unsigned)W::ALLOC) : "memory");
    }
}

template <class T, bool SPLIT, int NB, int NR> int prepare_shape() {
    IT_CUDA(cudaFuncSetAttribute(k_tree_attention_tc<T, SPLIT, NB, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTree<SPLIT, NB, NR>::TOTAL));
    // setmaxnreg deals out the registers of the launch: a kernel compiled to fewer would wait for ever
    cudaFuncAttributes at;
    IT_CUDA(cudaFuncGetAttributes(&at, k_tree_attention_tc<T, SPLIT, NB, NR>));
    using L = TcTree<SPLIT, NB, NR>;
    if (at.numRegs < L::REGS) return it_fail(IT_ESTATE, "it_tree_attention: built with %d registers a thread", at.numRegs);
    return IT_OK;
}
template <class T, bool SPLIT, int NB> int prepare_dim() {
    if (const int r = prepare_shape<T, SPLIT, NB, 16>()) return r;
    if (const int r = prepare_shape<T, SPLIT, NB, 32>()) return r;
    if (const int r = prepare_shape<T, SPLIT, NB, 64>()) return r;
    IT_CUDA(cudaFuncSetAttribute(k_tree_weights_tc<T, SPLIT, NB, TW_ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcWeights<SPLIT, NB, TW_ROWS>::TOTAL));
    return IT_OK;
}
template <class T, bool SPLIT> int prepare_type() { const int r = prepare_dim<T, SPLIT, 2>(); return r ? r : prepare_dim<T, SPLIT, 4>(); }

template <class T, bool SPLIT, int NB, int NR> int run_shape(const TaParams& p, int row_tiles, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    IT_CUDA(it_launch_early(k_tree_attention_tc<T, SPLIT, NB, NR>, dim3(p.splits, p.kv_heads, row_tiles), dim3(TcTree<SPLIT, NB, NR>::THREADS), TcTree<SPLIT, NB, NR>::TOTAL, st, p.joined ? p.splits : 1, km, vm, p));
    return IT_OK;
}
template <class T, bool SPLIT, int NB> int weigh_dim(const TaParams& p, const CUtensorMap& km, cudaStream_t st) {
    // one wave of CTAs, as many tiles for each
    const int tiles = (p.cached + p.rows + TA_KEYS - 1) / TA_KEYS, most = p.kv_heads < TA_MAXSPLITS ? TA_MAXSPLITS / p.kv_heads : 1, rounds = (tiles + most - 1) / most;
    IT_CUDA(it_launch_early(k_tree_weights_tc<T, SPLIT, NB, TW_ROWS>, dim3((tiles + rounds - 1) / rounds, p.kv_heads), dim3(TW_THREADS), TcWeights<SPLIT, NB, TW_ROWS>::TOTAL, st, 1, km, p));
    return IT_OK;
}
template <class T, bool SPLIT, int NB> int run_dim(const TaParams& p, int nr, int row_tiles, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    return nr == 16 ? run_shape<T, SPLIT, NB, 16>(p, row_tiles, km, vm, st) : nr == 32 ? run_shape<T, SPLIT, NB, 32>(p, row_tiles, km, vm, st) : run_shape<T, SPLIT, NB, 64>(p, row_tiles, km, vm, st);
}

}  // namespace

int it_tree_tc_prepare() {
    if (const int r = prepare_type<__half, true>()) return r;
    if (const int r = prepare_type<__half, false>()) return r;
    return prepare_type<__nv_bfloat16, false>();
}
int it_tree_tc_run(const TaParams& p, int type, int nb, int nr, int row_tiles, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    if (type == IT_F32) return nb <= 2 ? run_dim<__half, true, 2>(p, nr, row_tiles, km, vm, st) : run_dim<__half, true, 4>(p, nr, row_tiles, km, vm, st);
    if (type == IT_F16) return nb <= 2 ? run_dim<__half, false, 2>(p, nr, row_tiles, km, vm, st) : run_dim<__half, false, 4>(p, nr, row_tiles, km, vm, st);
    return nb <= 2 ? run_dim<__nv_bfloat16, false, 2>(p, nr, row_tiles, km, vm, st) : run_dim<__nv_bfloat16, false, 4>(p, nr, row_tiles, km, vm, st);
}
int it_tree_tc_weigh(const TaParams& p, int type, int nb, const CUtensorMap& km, cudaStream_t st) {
    if (type == IT_F32) return nb <= 2 ? weigh_dim<__half, true, 2>(p, km, st) : weigh_dim<__half, true, 4>(p, km, st);
    if (type == IT_F16) return nb <= 2 ? weigh_dim<__half, false, 2>(p, km, st) : weigh_dim<__half, false, 4>(p, km, st);
    return nb <= 2 ? weigh_dim<__nv_bfloat16, false, 2>(p, km, st) : weigh_dim<__nv_bfloat16, false, 4>(p, km, st);
}
