// Attention of a token, a chain or a tree of drafted tokens over a KV cache that the caller owns.  Stands where VkEngine records its attention
// dispatch (src/vk/mod.rs:833-840; CPU: src/cpu.rs:177-186), for any strides and lengths; sums are those of a softmax with a running maximum, not the
// reference's position order.
//
//   p = softmax(scale q.k) over the slots that a row sees,   out = (p v) * sigmoid(gate),   weights[g][slot] += sum of p over rows and heads of g
//
// One pass over K and V.  All rows and query heads of a KV head share its keys, so they are the rows of one matrix product ("product rows": row t * group + head); the
// cache is cut into runs of 64-slot tiles, one per CTA, so that a single token's few rows still use every SM, and k_tree_join puts the runs' sums together.
// A producer warp streams tiles with a tensor map (boxes of 64 slots x 64 elements, 128-byte swizzle: what ldmatrix reads without conflicts; slots behind the
// last one arrive as zeros) through a ring; consumer warps split a tile's product rows (WR) and slots (WK), every one with its own running maximum, sum and output
// in registers, joined at the end through shared memory.
// f32 activations: q (scaled per row by a power of two to the top of f16's range) and p (scaled by 2^14) are each the sum of two f16 values, 22 bits, and every product is
// done twice; the f16 cache is exact.  16-bit activations: p is rounded to the cache's type like the output itself, q is exact.
// Masks: only tiles that reach behind the cached slots look at them.  A masked score is replaced, whatever it was; there a non-finite V element is
// taken out of the product and added to the rows that do see it (0 * inf would be NaN in those that do not).
#include "it_tree_attention.cuh"
#include <mutex>

namespace {

// Shared memory: q (twice for f32 activations), then the ring of units (64 slots of K or of V), then the small things.
template <bool SPLIT, int NB, int R> struct TaSmem {
    static constexpr int QB = NB * R * 128, UNIT = NB * TA_KEYS * 128;
    static constexpr int Q = 0, RING = QB * (SPLIT ? 2 : 1);
    static constexpr int SMALL_BYTES = TA_MAXROWS * TA_WORDS * 4 + TA_MAXROWS * 4 + R * 4 + 16 * R * 8 + TA_UNIT_MAX * 16 + 64;
    static constexpr int FIT = (TA_SMEM_MAX - 1024 - SMALL_BYTES - RING) / UNIT;
    static constexpr int UNITS = FIT < TA_UNIT_MAX ? FIT : TA_UNIT_MAX;
    static constexpr int SMALL = RING + UNITS * UNIT;
    static constexpr int ANC = SMALL, JUMP = ANC + TA_MAXROWS * TA_WORDS * 4, FAC = JUMP + TA_MAXROWS * 4, ML = FAC + R * 4, BARS = ML + 16 * R * 8, FLAG = BARS + TA_UNIT_MAX * 16;
    static constexpr int TOTAL = FLAG + 64 + 1024;
    static_assert(UNITS >= 2, "K and V of a tile");
};

// Product rows [r0, r0 + R) of KV head g into shared memory, and for each the factor from the product to log2 of its exponential.
template <class T, bool SPLIT, int NB, int R>
__device__ void ta_load_q(const TaParams& p, unsigned char* smem, int g, int r0) {
    using L = TaSmem<SPLIT, NB, R>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    float* fac = reinterpret_cast<float*>(smem + L::FAC);
    for (int i = warp; i < R; i += nw) {
        const int r = r0 + i, t = r / p.group, h = g * p.group + r % p.group;
        const bool live = r < p.prows && 8 * lane < p.dim;
        unsigned hi[4] = {}, lo[4] = {};
        const float f = ta_q_row<T, SPLIT>(p, live, t, h, lane, hi, lo);
        if (lane < NB * 8) {
            const unsigned at = (unsigned)((lane >> 3) * R * 128) + swz(i, lane & 7);
            *reinterpret_cast<uint4*>(smem + L::Q + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) *reinterpret_cast<uint4*>(smem + L::Q + L::QB + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (lane == 0) fac[i] = f;
    }
}

// Products of the warp's 16 rows with KT of a tile's slots: s[n][..] of slots key0 + 8 n .. in the accumulator layout of mma.m16n8k16 (thread 4 g + t: rows g and
// g + 8, slots 2 t and 2 t + 1).
template <class T, bool SPLIT, int NB, int R, int KT>
__device__ __forceinline__ void ta_scores(float (&s)[KT / 8][4], unsigned q0, unsigned k0, int row0, int key0, int lane) {
    using L = TaSmem<SPLIT, NB, R>;
    const int li = lane >> 3, l8 = lane & 7;
    const int qr = row0 + l8 + (li & 1) * 8, qc = li >> 1, kr = key0 + l8 + (li >> 1) * 8, kc = li & 1;
    float s2[KT / 8][4];                        // every other step (f32 activations: the low halves), for more products in flight
#pragma unroll
    for (int n = 0; n < KT / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] = s2[n][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NB * 4; ks++) {
        unsigned a[4], al[4];
        const unsigned qa = q0 + (unsigned)((ks >> 2) * R * 128) + swz(qr, (ks & 3) * 2 + qc);
        ldsm4(a, qa);
        if constexpr (SPLIT) ldsm4(al, qa + L::QB);
#pragma unroll
        for (int n = 0; n < KT / 16; n++) {
            unsigned b[4];
            ldsm4(b, k0 + (unsigned)((ks >> 2) * TA_KEYS * 128) + swz(kr + 16 * n, (ks & 3) * 2 + kc));
            if constexpr (SPLIT) {
                Ta16<T>::mma(s[2 * n], a, b[0], b[1]); Ta16<T>::mma(s[2 * n + 1], a, b[2], b[3]);
                Ta16<T>::mma(s2[2 * n], al, b[0], b[1]); Ta16<T>::mma(s2[2 * n + 1], al, b[2], b[3]);
            } else if (ks & 1) { Ta16<T>::mma(s2[2 * n], a, b[0], b[1]); Ta16<T>::mma(s2[2 * n + 1], a, b[2], b[3]); }
            else { Ta16<T>::mma(s[2 * n], a, b[0], b[1]); Ta16<T>::mma(s[2 * n + 1], a, b[2], b[3]); }
        }
    }
#pragma unroll
    for (int n = 0; n < KT / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] += s2[n][i];
}

template <class T, bool SPLIT, int NB, int WR, int WK>
__global__ void __launch_bounds__(32 * (WR * WK + 1), 1)
k_tree_attention(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TaParams p) {
    constexpr int R = 16 * WR, KT = TA_KEYS / WK, HD = 64 * NB, NW = WR * WK;
    using L = TaSmem<SPLIT, NB, R>;
    using TA = typename std::conditional<SPLIT, float, T>::type;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, g = blockIdx.y, r0 = blockIdx.z * R;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::FLAG);
    const unsigned full0 = smem_u32(smem + L::BARS), empty0 = full0 + 8 * TA_UNIT_MAX, ring = smem_u32(smem + L::RING);
    unsigned (*anc)[TA_WORDS] = reinterpret_cast<unsigned (*)[TA_WORDS]>(smem + L::ANC);
    float* fac = reinterpret_cast<float*>(smem + L::FAC);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int cached = ta_cached(p), total = cached + p.rows, tiles = (total + TA_KEYS - 1) / TA_KEYS;
    const int tile0 = (int)((long long)split * tiles / p.splits), tile1 = (int)((long long)(split + 1) * tiles / p.splits);
    if (tid == 0) {
        *abort_flag = 0;
        for (int u = 0; u < L::UNITS; u++) { mbar_init(full0 + 8 * u, 1); mbar_init(empty0 + 8 * u, NW); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == NW && lane == 0) {            // the first units before anything else: their slots are free
        int n = 0;
        for (int tile = tile0; tile < tile1 && n < L::UNITS; tile++)
            for (int kv = 0; kv < 2 && n < L::UNITS; kv++, n++) {
                mbar_expect_tx(full0 + 8 * n, L::UNIT);
#pragma unroll
                for (int b = 0; b < NB; b++) tma_load_3d(ring + n * L::UNIT + b * TA_KEYS * 128, kv ? &vmap : &kmap, 64 * b, tile * TA_KEYS, g, full0 + 8 * n);
            }
    }
    ta_load_q<T, SPLIT, NB, R>(p, smem, g, r0);
    if (p.parents && tile1 * TA_KEYS > cached && tile0 < tile1) ta_ancestors(anc, reinterpret_cast<int*>(smem + L::JUMP), p.parents, p.rows);
    __syncthreads();

    float o[HD / 8][4];
    float m[2] = { -INFINITY, -INFINITY }, l[2] = { 0.f, 0.f };
#pragma unroll
    for (int n = 0; n < HD / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][i] = 0.f;
    const int wr = warp % WR, wk = warp / WR, row0 = 16 * wr, key0 = KT * wk, gg = lane >> 2, tt = lane & 3;
    bool ok = true;
    if (warp == NW) {
        // ---------------- producer: the units behind the first ring
        if (lane == 0) {
            int issued = 0, u = 0; unsigned ph = 0;
            const int units = 2 * (tile1 - tile0);
            for (int n = 0; n < units; n++) {
                if (n >= L::UNITS) {
                    if (!mbar_wait(empty0 + 8 * u, ph ^ 1u, abort_flag, p.status, 41)) break;
                    mbar_expect_tx(full0 + 8 * u, L::UNIT);
#pragma unroll
                    for (int b = 0; b < NB; b++)
                        tma_load_3d(ring + u * L::UNIT + b * TA_KEYS * 128, (n & 1) ? &vmap : &kmap, 64 * b, (tile0 + (n >> 1)) * TA_KEYS, g, full0 + 8 * u);
                }
                issued = n + 1;
                if (++u == L::UNITS) { u = 0; ph ^= 1u; }
            }
            if (*abort_flag) {                 // leave only after every copy has landed (bounded)
                for (int k = issued > L::UNITS ? issued - L::UNITS : 0; k < issued; k++) {
                    const long long t0 = clock64();
                    while (!mbar_test(full0 + 8 * (k % L::UNITS), (unsigned)(k / L::UNITS) & 1u) && clock64() - t0 < WAIT_CLOCKS) { }
                }
            }
        }
    } else {
        const float f[2] = { fac[row0 + gg], fac[row0 + gg + 8] };
        const int t0 = min((r0 + row0 + gg) / p.group, p.rows - 1), t1 = min((r0 + row0 + gg + 8) / p.group, p.rows - 1);
        const unsigned q0 = smem_u32(smem + L::Q);
        const int li = lane >> 3, l8 = lane & 7;
        int u = 0; unsigned ph = 0;
        for (int tile = tile0; tile < tile1; tile++) {
            ok = ok && mbar_wait_warp(full0 + 8 * u, ph, abort_flag, p.status, 42);
            if (!ok) break;
            float s[KT / 8][4];
            ta_scores<T, SPLIT, NB, R, KT>(s, q0, ring + u * L::UNIT, row0, key0, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * u);
            if (++u == L::UNITS) { u = 0; ph ^= 1u; }
            const bool masked = (tile + 1) * TA_KEYS > cached;
            float mx[2] = { -INFINITY, -INFINITY };
#pragma unroll
            for (int n = 0; n < KT / 8; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[n][i] *= f[i >> 1];
                    if (masked && !ta_sees(p, anc, i >> 1 ? t1 : t0, tile * TA_KEYS + key0 + 8 * n + 2 * tt + (i & 1), cached)) s[n][i] = -INFINITY;
                    mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
                }
            float base[2], corr[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                const float mn = fmaxf(m[i], mx[i]), ref = mn == -INFINITY ? 0.f : mn;
                corr[i] = ex2(m[i] - ref); base[i] = ref - TA_SHIFT; m[i] = mn; l[i] *= corr[i];
            }
            if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                for (int n = 0; n < HD / 8; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][i] *= corr[i >> 1];
            }
            unsigned ph_[KT / 16][4], pl[KT / 16][4];
#pragma unroll
            for (int n = 0; n < KT / 8; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++) { s[n][i] = ex2(s[n][i] - base[i >> 1]); l[i >> 1] += s[n][i]; }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const unsigned h = Ta16<T>::pack(s[n][2 * i], s[n][2 * i + 1]);
                    ph_[n >> 1][(n & 1) * 2 + i] = h;
                    if constexpr (SPLIT) { const float2 b = Ta16<T>::unpack(h); pl[n >> 1][(n & 1) * 2 + i] = Ta16<T>::pack(s[n][2 * i] - b.x, s[n][2 * i + 1] - b.y); }
                }
            }
            ok = mbar_wait_warp(full0 + 8 * u, ph, abort_flag, p.status, 43);
            if (!ok) break;
            const unsigned v0 = ring + u * L::UNIT;
            bool odd = false;
#pragma unroll
            for (int c = 0; c < KT / 16; c++) {
                const int vr = key0 + 16 * c + l8 + (li & 1) * 8;
#pragma unroll
                for (int n = 0; n < HD / 16; n++) {
                    unsigned b[4];
                    ldsm4t(b, v0 + (unsigned)((n >> 2) * TA_KEYS * 128) + swz(vr, (n & 3) * 2 + (li >> 1)));
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 4; i++) b[i] = finite_only<T>(b[i], odd);
                    }
                    Ta16<T>::mma(o[2 * n], ph_[c], b[0], b[1]); Ta16<T>::mma(o[2 * n + 1], ph_[c], b[2], b[3]);
                    if constexpr (SPLIT) { Ta16<T>::mma(o[2 * n], pl[c], b[0], b[1]); Ta16<T>::mma(o[2 * n + 1], pl[c], b[2], b[3]); }
                }
            }
            if (masked && __any_sync(0xffffffffu, odd)) {      // rare: what was taken out goes to the rows that see its slot
                const unsigned char* v = smem + L::RING + u * L::UNIT;
                for (int k = key0; k < key0 + KT; k++) {
                    const int j = tile * TA_KEYS + k;
                    const bool see0 = ta_sees(p, anc, t0, j, cached), see1 = ta_sees(p, anc, t1, j, cached);
#pragma unroll
                    for (int n = 0; n < HD / 8; n++) {
                        const unsigned raw = *reinterpret_cast<const unsigned*>(v + (n >> 3) * TA_KEYS * 128 + swz(k, n & 7) + 4 * tt);
                        const float2 x = Ta16<T>::unpack(raw);
                        const bool nx = (raw & Ta16<T>::EXP) == Ta16<T>::EXP, ny = ((raw >> 16) & Ta16<T>::EXP) == Ta16<T>::EXP;
                        if (see0 && nx) o[n][0] += x.x;
                        if (see0 && ny) o[n][1] += x.y;
                        if (see1 && nx) o[n][2] += x.x;
                        if (see1 && ny) o[n][3] += x.y;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * u);
            if (++u == L::UNITS) { u = 0; ph ^= 1u; }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
    }
    __syncwarp();
    __syncthreads();                           // every copy has been read: the ring is free
    // ---------------- the warps that share rows join: the first one's accumulators take in the others'
    float2* ml = reinterpret_cast<float2*>(smem + L::ML);           // [WK][R]
    float* jo = reinterpret_cast<float*>(smem + L::RING);           // [WK - 1][R][HD]
    static_assert((WK - 1) * R * HD * 4 <= L::UNITS * L::UNIT, "the ring holds the other warps' accumulators");
    const bool bad = *abort_flag != 0;
    if (warp < NW && tt == 0) { ml[wk * R + row0 + gg] = make_float2(m[0], l[0]); ml[wk * R + row0 + gg + 8] = make_float2(m[1], l[1]); }
    __syncthreads();
    float sc[2] = { 1.f, 1.f }, mf[2], lf[2] = { 0.f, 0.f };
    if (warp < NW) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mf[i] = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; k++) mf[i] = fmaxf(mf[i], ml[k * R + row0 + gg + 8 * i].x);
            const float ref = mf[i] == -INFINITY ? 0.f : mf[i];
#pragma unroll
            for (int k = 0; k < WK; k++) { const float2 e = ml[k * R + row0 + gg + 8 * i]; lf[i] += e.y * ex2(e.x - ref); }
            sc[i] = ex2(m[i] - ref);
        }
#pragma unroll
        for (int n = 0; n < HD / 8; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                o[n][2 * i] *= sc[i]; o[n][2 * i + 1] *= sc[i];
                if (wk > 0) *reinterpret_cast<float2*>(jo + ((size_t)(wk - 1) * R + row0 + gg + 8 * i) * HD + ((8 * n + 2 * tt) ^ (8 * (gg & 3)))) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
    }
    __syncthreads();
    if (warp >= WR) return;
#pragma unroll
    for (int k = 0; k < WK - 1; k++)
#pragma unroll
        for (int n = 0; n < HD / 8; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 e = *reinterpret_cast<const float2*>(jo + ((size_t)k * R + row0 + gg + 8 * i) * HD + ((8 * n + 2 * tt) ^ (8 * (gg & 3))));
                o[n][2 * i] += e.x; o[n][2 * i + 1] += e.y;
            }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = r0 + row0 + gg + 8 * i;
        if (r >= p.prows) continue;
        const float lsum = bad ? NAN : lf[i];
        if (p.splits > 1) {
            const size_t at = ((size_t)split * p.kv_heads + g) * p.pad_rows + r;
            if (tt == 0) p.part_ml[at] = make_float2(mf[i] == -INFINITY ? -INFINITY : mf[i] - TA_SHIFT, lsum);
            if (mf[i] == -INFINITY && !bad && lsum == 0.f) continue;            // nothing seen: not read either
#pragma unroll
            for (int n = 0; n < HD / 8; n++) __stcg(reinterpret_cast<float2*>(p.part_o + at * HD + 8 * n + 2 * tt), make_float2(o[n][2 * i], o[n][2 * i + 1]));
        } else {
            const int t = r / p.group, h = g * p.group + r % p.group;
            if (p.stats && tt == 0) p.stats[(size_t)g * p.pad_rows + r] = make_float2(mf[i] == -INFINITY ? 0.f : mf[i] - TA_SHIFT, lsum);
            const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
            TA* out = (TA*)p.out + t * p.o_row + h * p.o_head;
            const TA* gate = p.gate ? (const TA*)p.gate + t * p.g_row + h * p.g_head : nullptr;
#pragma unroll
            for (int n = 0; n < HD / 8; n++) {
                const int c = 8 * n + 2 * tt;
                if (c >= p.dim) continue;
                float x = o[n][2 * i] * inv, y = o[n][2 * i + 1] * inv;
                if (gate) { x /= 1.f + __expf(-to_f32(gate[c])); y /= 1.f + __expf(-to_f32(gate[c + 1])); }
                out[c] = from_f32<TA>(x); out[c + 1] = from_f32<TA>(y);
            }
        }
    }
}

// Joins the runs of one product row: out = sum of the runs' outputs, each scaled to the common maximum, over the sum of their sums.  Four groups of HD / 4 threads
// take every fourth run; runs that saw nothing are not read.
template <class TA, int NB>
__global__ void __launch_bounds__(64 * NB) k_tree_join(const __grid_constant__ TaParams p) {
    constexpr int HD = 64 * NB, LANES = HD / 4;
    __shared__ float wgt[1024];
    __shared__ float red[2][32];
    __shared__ float4 acc[3][LANES];
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, r = blockIdx.x, g = blockIdx.y, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
    const size_t step = (size_t)p.kv_heads * p.pad_rows, at = (size_t)g * p.pad_rows + r;
    float top = -INFINITY;
    for (int s = tid; s < p.splits; s += blockDim.x) top = fmaxf(top, __ldcg(&p.part_ml[s * step + at]).x);
#pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
    for (int k = 0; k < nw; k++) top = fmaxf(top, red[0][k]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int s = tid; s < p.splits; s += blockDim.x) {
        const float2 e = __ldcg(&p.part_ml[s * step + at]);
        const float w = ex2(e.x - ref);
        wgt[s] = e.x == -INFINITY && e.y == 0.f ? -1.f : w;           // -1: not written, not read
        sum += e.y * w;
    }
    // a fixed order, so that the same inputs give the same bits
#pragma unroll
    for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0) red[1][warp] = sum;
    __syncthreads();
    sum = 0.f;
    for (int k = 0; k < nw; k++) sum += red[1][k];
    const int grp = tid / LANES, c = tid % LANES * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = grp; s < p.splits; s += 4) {
        const float w = wgt[s];
        if (w < 0.f) continue;
        const float4 e = __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * step + at) * HD + c));
        a.x = fmaf(w, e.x, a.x); a.y = fmaf(w, e.y, a.y); a.z = fmaf(w, e.z, a.z); a.w = fmaf(w, e.w, a.w);
    }
    if (grp) acc[grp - 1][tid % LANES] = a;
    __syncthreads();
    if (p.stats && tid == 0) p.stats[at] = make_float2(ref, sum);
    if (grp || c >= p.dim) return;
#pragma unroll
    for (int k = 0; k < 3; k++) { const float4 e = acc[k][tid]; a.x += e.x; a.y += e.y; a.z += e.z; a.w += e.w; }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int t = r / p.group, h = g * p.group + r % p.group;
    float v[4] = { a.x * inv, a.y * inv, a.z * inv, a.w * inv };
    if (p.gate) {
        float z[4]; load4((const TA*)p.gate + t * p.g_row + h * p.g_head + c, z);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] /= 1.f + __expf(-z[i]);
    }
    store4((TA*)p.out + t * p.o_row + h * p.o_head + c, v);
}

// Received weight: the scores of a 64-slot tile once more, against the finished maximum and sum of every product row, summed down the columns.  One CTA has a tile of
// a KV head and all rows, so no sum crosses CTAs and its order is fixed.
template <class T, bool SPLIT, int NB, int WR, int WK>
__global__ void __launch_bounds__(32 * WR * WK)
k_tree_weights(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ TaParams p) {
    constexpr int R = 16 * WR, KT = TA_KEYS / WK;
    using L = TaSmem<SPLIT, NB, R>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tile = blockIdx.x, g = blockIdx.y;
    const int cached = ta_cached(p), total = cached + p.rows;
    if (tile * TA_KEYS >= total) { asm volatile("griddepcontrol.wait;" ::: "memory"); return; }
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::FLAG);
    const unsigned full0 = smem_u32(smem + L::BARS), ring = smem_u32(smem + L::RING);
    unsigned (*anc)[TA_WORDS] = reinterpret_cast<unsigned (*)[TA_WORDS]>(smem + L::ANC);
    float* fac = reinterpret_cast<float*>(smem + L::FAC);
    float* col = reinterpret_cast<float*>(smem + L::ML);           // [WR][64]
    if (tid == 0) {
        *abort_flag = 0; mbar_init(full0, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(full0, L::UNIT);
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_3d(ring + b * TA_KEYS * 128, &kmap, 64 * b, tile * TA_KEYS, g, full0);
    }
    const bool masked = (tile + 1) * TA_KEYS > cached;
    if (masked && p.parents) ta_ancestors(anc, reinterpret_cast<int*>(smem + L::JUMP), p.parents, p.rows);
    asm volatile("griddepcontrol.wait;" ::: "memory");             // the statistics come from the kernel before
    __syncthreads();
    const int wr = warp % WR, wk = warp / WR, row0 = 16 * wr, key0 = KT * wk, gg = lane >> 2, tt = lane & 3;
    float sum[KT / 8][2];
#pragma unroll
    for (int n = 0; n < KT / 8; n++) sum[n][0] = sum[n][1] = 0.f;
    const bool ok = mbar_wait_warp(full0, 0, abort_flag, p.status, 44);
    for (int r0 = 0; r0 < p.prows; r0 += R) {
        ta_load_q<T, SPLIT, NB, R>(p, smem, g, r0);
        __syncthreads();
        float s[KT / 8][4];
        ta_scores<T, SPLIT, NB, R, KT>(s, smem_u32(smem + L::Q), ring, row0, key0, lane);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = r0 + row0 + gg + 8 * i;
            if (r >= p.prows) continue;
            const float f = fac[row0 + gg + 8 * i];
            const float2 st = __ldcg(&p.stats[(size_t)g * p.pad_rows + r]);
            const float inv = st.y == 0.f ? 0.f : 1.f / st.y;
            const int t = r / p.group;
#pragma unroll
            for (int n = 0; n < KT / 8; n++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    if (!masked || ta_sees(p, anc, t, tile * TA_KEYS + key0 + 8 * n + 2 * tt + c, cached)) sum[n][c] += ex2(s[n][2 * i + c] * f - st.x) * inv;
        }
        __syncthreads();                       // before the next rows take the place of these
    }
#pragma unroll
    for (int n = 0; n < KT / 8; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float v = sum[n][c];
            v += __shfl_xor_sync(0xffffffffu, v, 4); v += __shfl_xor_sync(0xffffffffu, v, 8); v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (gg == 0) col[wr * TA_KEYS + key0 + 8 * n + 2 * tt + c] = v;
        }
    __syncthreads();
    if (tid < TA_KEYS && tile * TA_KEYS + tid < total) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WR; k++) v += col[k * TA_KEYS + tid];
        float* w = p.weights + (long long)g * p.w_head + tile * TA_KEYS + tid;
        *w = ok ? *w + v : NAN;
    }
    if (!ok && tid == 0) {                     // leave only after the copy has landed (bounded)
        const long long t0 = clock64();
        while (!mbar_test(full0, 0) && clock64() - t0 < WAIT_CLOCKS) { }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
// How a call is cut: rows of a CTA's product tile, tiles of product rows, runs of the cache.
struct TaPlan { bool tc; int nb, wr, nr, pad_rows, row_tiles, splits; size_t part_o, part_ml, stats, total; };

// Which kernel: see the figures at the rule.  IT_TREE=mma|tc forces one (for tests and measurements).
bool ta_takes_tc(int prows, long slots) {
    if (const char* v = getenv("IT_TREE")) return v[0] == 't';
    return true;
}

TaPlan ta_plan(const it_tree_attention_args* a, int sm_count) {
    TaPlan pl;
    const int group = a->heads / a->kv_heads, prows = a->rows * group;
    pl.tc = ta_takes_tc(prows, (long)a->cached + a->rows);
    pl.nb = a->head_dim <= 64 && !pl.tc ? 1 : a->head_dim <= 128 ? 2 : 4;
    // mma.sync: four consumer warps (with the producer five: two on one sub-core, which leaves a thread 255 registers; nine warps leave it 168 and spill): 16 product rows each
    // share the rows and split a tile's slots, 32: two by two, 64: a warp for 16 rows
    pl.wr = prows <= 16 ? 1 : prows <= 32 ? 2 : 4;
    pl.nr = 16 * pl.wr;
    pl.row_tiles = (prows + pl.nr - 1) / pl.nr;
    pl.pad_rows = pl.row_tiles * pl.nr;
    const long keys = pl.tc ? 128 : TA_KEYS, tiles = ((long)a->cached + a->rows + keys - 1) / keys, ctas = (long)a->kv_heads * pl.row_tiles;
    long splits = sm_count / ctas;             // one wave of CTAs
    if (splits > tiles) splits = tiles;
    if (splits < 1) splits = 1;
    pl.splits = (int)splits;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = (size_t)a->kv_heads * pl.pad_rows;
    pl.part_o = 0;
    pl.part_ml = splits > 1 ? up((size_t)splits * rows * 64 * pl.nb * 4) : 0;
    pl.stats = pl.part_ml + (splits > 1 ? up((size_t)splits * rows * 8) : 0);
    pl.total = pl.stats + up(rows * 8);        // the statistics of a call without weights are not kept, but sizes do not depend on pointers
    return pl;
}

typedef CUresult (*ta_encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int ta_map(CUtensorMap* map, const void* cache, int type, int dim, int64_t slots, int64_t slot, int heads, int64_t head, int keys) {
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
    const cuuint32_t box[3] = { 64, (cuuint32_t)keys, 1 }, estr[3] = { 1, 1, 1 };
    const CUresult r = encode(map, type == IT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(cache), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? IT_OK : it_fail(IT_ECUDA, "it_tree_attention: cuTensorMapEncodeTiled failed with code %d", (int)r);
}

// Shared-memory limits of every kernel, set (and the kernels loaded) by the first call on a device, so that later calls can be recorded.
template <class F> int ta_set(F f, int bytes) { IT_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)); return IT_OK; }
template <class T, bool SPLIT, int NB, int WR, int WK> int ta_prepare_shape() {
    using L = TaSmem<SPLIT, NB, 16 * WR>;
    if (const int r = ta_set(k_tree_attention<T, SPLIT, NB, WR, WK>, L::TOTAL)) return r;
    return ta_set(k_tree_weights<T, SPLIT, NB, WR, WK>, L::TOTAL);
}
template <class T, bool SPLIT, int NB> int ta_prepare_dim() {
    if (const int r = ta_prepare_shape<T, SPLIT, NB, 1, 4>()) return r;
    if (const int r = ta_prepare_shape<T, SPLIT, NB, 2, 2>()) return r;
    if (const int r = ta_prepare_shape<T, SPLIT, NB, 4, 1>()) return r;
    cudaFuncAttributes at;
    IT_CUDA(cudaFuncGetAttributes(&at, k_tree_join<typename std::conditional<SPLIT, float, T>::type, NB>));
    return IT_OK;
}
template <class T, bool SPLIT> int ta_prepare_type() {
    if (const int r = ta_prepare_dim<T, SPLIT, 1>()) return r;
    if (const int r = ta_prepare_dim<T, SPLIT, 2>()) return r;
    return ta_prepare_dim<T, SPLIT, 4>();
}
int ta_prepare(int device) {
    static std::mutex lock; static bool done[64] = {};
    std::lock_guard<std::mutex> hold(lock);
    if (done[device]) return IT_OK;
    if (const int r = ta_prepare_type<__half, true>()) return r;
    if (const int r = ta_prepare_type<__half, false>()) return r;
    if (const int r = ta_prepare_type<__nv_bfloat16, false>()) return r;
    if (const int r = it_tree_tc_prepare()) return r;
    done[device] = true;
    return IT_OK;
}

int ta_join(const TaParams& p, int type, int nb, cudaStream_t st) {
    const dim3 grid(p.prows, p.kv_heads), block(64 * nb);
    auto go = [&](auto kern) -> int { IT_CUDA(ta_launch(true, kern, grid, block, 0, st, p)); return IT_OK; };
    if (type == IT_F32) return nb == 1 ? go(k_tree_join<float, 1>) : nb == 2 ? go(k_tree_join<float, 2>) : go(k_tree_join<float, 4>);
    if (type == IT_F16) return nb == 1 ? go(k_tree_join<__half, 1>) : nb == 2 ? go(k_tree_join<__half, 2>) : go(k_tree_join<__half, 4>);
    return nb == 1 ? go(k_tree_join<__nv_bfloat16, 1>) : nb == 2 ? go(k_tree_join<__nv_bfloat16, 2>) : go(k_tree_join<__nv_bfloat16, 4>);
}
template <class T, bool SPLIT, int NB, int WR, int WK>
int ta_run(const TaParams& p, const TaPlan& pl, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    using L = TaSmem<SPLIT, NB, 16 * WR>;
    using TA = typename std::conditional<SPLIT, float, T>::type;
    IT_CUDA(ta_launch(false, k_tree_attention<T, SPLIT, NB, WR, WK>, dim3(pl.splits, p.kv_heads, pl.row_tiles), dim3(32 * (WR * WK + 1)), L::TOTAL, st, km, vm, p));
    if (pl.splits > 1) IT_CUDA(ta_launch(true, k_tree_join<TA, NB>, dim3(p.prows, p.kv_heads), dim3(64 * NB), 0, st, p));
    if (p.weights) IT_CUDA(ta_launch(true, k_tree_weights<T, SPLIT, NB, WR, WK>, dim3((p.cached + p.rows + TA_KEYS - 1) / TA_KEYS, p.kv_heads), dim3(32 * WR * WK), L::TOTAL, st, km, p));
    return IT_OK;
}
template <class T, bool SPLIT, int NB> int ta_run_dim(const TaParams& p, const TaPlan& pl, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    return pl.wr == 1 ? ta_run<T, SPLIT, NB, 1, 4>(p, pl, km, vm, st) : pl.wr == 2 ? ta_run<T, SPLIT, NB, 2, 2>(p, pl, km, vm, st) : ta_run<T, SPLIT, NB, 4, 1>(p, pl, km, vm, st);
}
template <class T, bool SPLIT> int ta_run_type(const TaParams& p, const TaPlan& pl, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    return pl.nb == 1 ? ta_run_dim<T, SPLIT, 1>(p, pl, km, vm, st) : pl.nb == 2 ? ta_run_dim<T, SPLIT, 2>(p, pl, km, vm, st) : ta_run_dim<T, SPLIT, 4>(p, pl, km, vm, st);
}

int ta_check_sizes(const it_tree_attention_args* a) {
    const char* const who = "it_tree_attention";
    IT_CHECK_ARG(a, "%s: null argument", who);
    IT_CHECK_ARG(it_type_pair(a->type, a->cache_type), "%s: types %d over %d", who, a->type, a->cache_type);
    IT_CHECK_ARG(a->rows >= 0 && a->rows <= TA_MAXROWS, "%s: %d rows, at most %d", who, a->rows, TA_MAXROWS);
    IT_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, "%s: head dimension %d is not a multiple of 8 up to 256", who, a->head_dim);
    IT_CHECK_ARG(a->kv_heads >= 1 && a->kv_heads <= 4096 && a->heads >= 1 && a->heads <= 16384 && a->heads % a->kv_heads == 0, "%s: %d heads over %d kv heads", who, a->heads, a->kv_heads);
    IT_CHECK_ARG(a->cached >= 0 && a->cached < ((int64_t)1 << 30), "%s: %lld cached slots", who, (long long)a->cached);
    return IT_OK;
}

}  // namespace

IT_API int it_tree_attention_workspace(const it_tree_attention_args* a, size_t* nbytes) {
    if (const int r = ta_check_sizes(a)) return r;
    IT_CHECK_ARG(nbytes, "it_tree_attention_workspace: null argument");
    // without a device: as many SMs as sm_100a parts have
    *nbytes = a->rows ? ta_plan(a, 148).total : 0;
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
    // the received weights read q again after out is written
    IT_CHECK_ARG((same(a->q, a->q_row, a->q_head) && !a->weights) || !it_overlap(a->q, it_span(T, a->q_row, H, a->q_head, D, es), a->out, os), "%s: out overlaps q", who);
    IT_CHECK_ARG(!a->gate || same(a->gate, a->g_row, a->g_head) || !it_overlap(a->gate, it_span(T, a->g_row, H, a->g_head, D, es), a->out, os), "%s: out overlaps gate", who);
    it_ops_device dev;
    if (const int r = it_ops_current(stream, who, &dev)) return r;
    if (const int r = ta_prepare(dev.device)) return r;
    const TaPlan pl = ta_plan(a, 148);
    IT_CHECK_ARG(a->workspace && it_aligned(a->workspace, 256) && a->workspace_bytes >= pl.total, "%s: a workspace of %zu bytes, 256-byte aligned, is needed", who, pl.total);
    CUtensorMap km, vm;
    if (const int r = ta_map(&km, a->k_cache, a->cache_type, a->head_dim, a->cached + T, a->kc_slot, a->kv_heads, a->kc_head, pl.tc ? 128 : TA_KEYS)) return r;
    if (const int r = ta_map(&vm, a->v_cache, a->cache_type, a->head_dim, a->cached + T, a->vc_slot, a->kv_heads, a->vc_head, pl.tc ? 128 : TA_KEYS)) return r;
    TaParams p;
    char* ws = (char*)a->workspace;
    p.q = a->q; p.gate = a->gate; p.out = a->out; p.parents = a->parents; p.length = a->length; p.weights = a->weights;
    p.part_o = (float*)(ws + pl.part_o); p.part_ml = (float2*)(ws + pl.part_ml); p.stats = a->weights ? (float2*)(ws + pl.stats) : nullptr; p.status = dev.status_dev;
    p.q_row = a->q_row; p.q_head = a->q_head; p.g_row = a->g_row; p.g_head = a->g_head; p.o_row = a->o_row; p.o_head = a->o_head; p.w_head = a->w_head;
    p.rows = a->rows; p.heads = a->heads; p.group = a->heads / a->kv_heads; p.kv_heads = a->kv_heads; p.dim = a->head_dim; p.cached = (int)a->cached; p.splits = pl.splits;
    p.prows = a->rows * p.group; p.pad_rows = pl.pad_rows; p.scale = a->scale == 0.f ? 1.f / sqrtf((float)a->head_dim) : a->scale;
    const cudaStream_t st = (cudaStream_t)stream;
    if (pl.tc) {
        if (const int r = it_tree_tc_run(p, a->type, pl.nb, pl.nr, pl.row_tiles, km, vm, st)) return r;
        if (p.splits > 1) if (const int r = ta_join(p, a->type, pl.nb, st)) return r;
        return p.weights ? it_tree_tc_weigh(p, a->type, pl.nb, pl.nr, km, st) : IT_OK;
    }
    if (a->type == IT_F32) return ta_run_type<__half, true>(p, pl, km, vm, st);
    if (a->type == IT_F16) return ta_run_type<__half, false>(p, pl, km, vm, st);
    return ta_run_type<__nv_bfloat16, false>(p, pl, km, vm, st);
}
