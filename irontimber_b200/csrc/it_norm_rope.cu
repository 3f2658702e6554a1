// Norms of q and k per head, rotation to positions, and the cache store, in one pass over a projection's rows.  Stands where VkEngine records
// its head norm, rope and kv-store dispatches (src/vk/mod.rs:815-832; CPU: src/cpu.rs:139-176), for a cache that the caller owns.
//
//   x' = x * (mean(x^2) + eps)^(-1/2) * w,   (a, b) of pair i -> m (a cos - b sin, a sin + b cos),   angle = position * f_i
//
// Angles: f_i is kept as a 64-bit fraction of a turn, so position * f_i modulo one turn is one integer product, exact for any position; its top 32 bits
// as a fraction of half a turn go to sincospi.  In f32 radians a position of 120,000 would already be off by 4e-3.
// What bounds it: bytes (4096 rows of 24 + 4 + 4 heads of 256, f32: 251 MB in 45 us, 0.87 of the measured copy rate), and for few rows the launch (2.5 us).  A warp has one head of one
// row in registers (two loads of four elements a lane), the next one on its way; the pairs of the rotation lie in other lanes
// and meet in the warp's own shared memory.  The table of a row's sines and cosines is made once by the CTA for its heads.
#include "it_ops.cuh"
#include <cmath>
#include <new>

struct it_rope { int n_rot, layout; double freq[128], mscale; unsigned long long turns[128]; };

namespace {

constexpr int NR_WARPS = 8, NR_MAXDIM = 256, NR_MAXPAIRS = NR_MAXDIM / 2;

struct NrParams {
    const void *q, *k, *v; void *q_out, *k_cache, *v_cache;
    long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, kc_slot, kc_head, vc_slot, vc_head, slots, slot0;
    const int *positions, *base; const float *q_norm, *k_norm;
    int rows, heads, kv_heads, dim, pos0, pairs, interleaved; float eps, mscale;
    unsigned long long turns[NR_MAXPAIRS];
};

// sin and cos of `turn` / 2^64 turns.  The 32 bits that are kept are a step of 1.5e-9 radians; their conversion rounds to 24 bits.
__device__ __forceinline__ void turn_sincos(unsigned long long turn, float* s, float* c) {
    sincospif((float)(int)(unsigned)(turn >> 32) * 4.656612873077392578125e-10f, s, c);
}

template <class TA, class TC>
__global__ void __launch_bounds__(NR_WARPS * 32) k_norm_rope(const __grid_constant__ NrParams p) {
    __shared__ float buf[NR_WARPS][NR_MAXDIM];
    __shared__ float2 table[NR_MAXPAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.x;
    const int nq = p.q ? p.heads : 0, nkv = p.k ? p.kv_heads : 0, step = NR_WARPS * gridDim.y;
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const int add = p.base ? *p.base : 0;
    const long long slot = p.slot0 + add + t;
    const int jobs = nkv && slot >= 0 && slot < p.slots ? nq + 2 * nkv : nq;       // k and v heads of a row without a slot are left out
    const bool lo = 4 * lane < p.dim, hi = 4 * lane + 128 < p.dim;
    // this row's heads, k heads, v heads; a lane has elements 4 lane .. and 128 + 4 lane ..
    const TA* const q = (const TA*)p.q + t * p.q_row + 4 * lane;
    const TA* const k = (const TA*)p.k + t * p.k_row + 4 * lane;
    const TA* const v = (const TA*)p.v + t * p.v_row + 4 * lane;
    float x[2][4];
    auto load = [&](int job) {
        const TA* s = job < nq ? q + job * p.q_head : job < nq + nkv ? k + (job - nq) * p.k_head : v + (job - nq - nkv) * p.v_head;
        if (lo) load4(s, x[0]);
        if (hi) load4(s + 128, x[1]);
    };
#pragma unroll
    for (int j = 0; j < 2; j++) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
    int job = blockIdx.y * NR_WARPS + warp;
    if (job < jobs) load(job);                 // under way while the table is made
    if (p.pairs) {
        const int pos = p.positions ? p.positions[t] : p.pos0 + add + t;
        for (int i = threadIdx.x; i < p.pairs; i += NR_WARPS * 32) {
            float s, c; turn_sincos((unsigned long long)(long long)pos * p.turns[i], &s, &c);
            table[i] = make_float2(c * p.mscale, s * p.mscale);
        }
        __syncthreads();
    }
    const float inv_dim = 1.0f / (float)p.dim;
    float* const b = buf[warp];
    for (; job < jobs; job += step) {
        float y[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) y[j][i] = x[j][i];
        if (job + step < jobs) load(job + step);                   // the next head while this one is worked on
        const bool is_q = job < nq;
        if (job < nq + nkv) {
            const float* w = is_q ? p.q_norm : p.k_norm;
            if (w) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s = fmaf(y[j][i], y[j][i], s);
#pragma unroll
                for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
                const float r = 1.0f / sqrtf(fmaf(s, inv_dim, p.eps));
                float u[4];
                if (lo) {
                    load4(w + 4 * lane, u);
#pragma unroll
                    for (int i = 0; i < 4; i++) y[0][i] *= r * u[i];
                }
                if (hi) {
                    load4(w + 4 * lane + 128, u);
#pragma unroll
                    for (int i = 0; i < 4; i++) y[1][i] *= r * u[i];
                }
            }
            if (p.pairs) {
                // the pairs lie in other lanes: through the warp's own memory.  A group of four may end behind the rotated part: those values come back as they went.
                const bool rlo = 4 * lane < 2 * p.pairs, rhi = 4 * lane + 128 < 2 * p.pairs;
                if (rlo) *reinterpret_cast<float4*>(b + 4 * lane) = make_float4(y[0][0], y[0][1], y[0][2], y[0][3]);
                if (rhi) *reinterpret_cast<float4*>(b + 4 * lane + 128) = make_float4(y[1][0], y[1][1], y[1][2], y[1][3]);
                __syncwarp();
                for (int i = lane; i < p.pairs; i += 32) {
                    const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + p.pairs;
                    const float2 cs = table[i]; const float a0 = b[ia], b0 = b[ib];
                    b[ia] = a0 * cs.x - b0 * cs.y; b[ib] = a0 * cs.y + b0 * cs.x;
                }
                __syncwarp();
                if (rlo) { const float4 a = *reinterpret_cast<const float4*>(b + 4 * lane); y[0][0] = a.x; y[0][1] = a.y; y[0][2] = a.z; y[0][3] = a.w; }
                if (rhi) { const float4 a = *reinterpret_cast<const float4*>(b + 4 * lane + 128); y[1][0] = a.x; y[1][1] = a.y; y[1][2] = a.z; y[1][3] = a.w; }
                __syncwarp();                  // before the next head's values take their place
            }
        }
        if (is_q) {
            TA* o = (TA*)p.q_out + t * p.qo_row + job * p.qo_head + 4 * lane;
            if (lo) store4(o, y[0]);
            if (hi) store4(o + 128, y[1]);
        } else {
            TC* o = (job < nq + nkv ? (TC*)p.k_cache + slot * p.kc_slot + (job - nq) * p.kc_head : (TC*)p.v_cache + slot * p.vc_slot + (job - nq - nkv) * p.vc_head) + 4 * lane;
            if (lo) store4(o, y[0]);
            if (hi) store4(o + 128, y[1]);
        }
    }
}

}  // namespace

IT_API int it_rope_create(const it_rope_config* c, it_rope** out) {
    IT_CHECK_ARG(c && out, "it_rope_create: null argument");
    *out = nullptr;
    IT_CHECK_ARG(c->n_rot >= 2 && c->n_rot <= NR_MAXDIM && c->n_rot % 2 == 0, "it_rope_create: n_rot %d is not an even number from 2 to 256", c->n_rot);
    IT_CHECK_ARG(c->layout == IT_ROPE_HALF || c->layout == IT_ROPE_INTERLEAVED, "it_rope_create: layout %d", c->layout);
    IT_CHECK_ARG(c->scaling >= IT_ROPE_SCALE_NONE && c->scaling <= IT_ROPE_SCALE_YARN, "it_rope_create: scaling %d", c->scaling);
    IT_CHECK_ARG(std::isfinite(c->base) && c->base > 1.0, "it_rope_create: base must be above 1");
    const bool scaled = c->scaling != IT_ROPE_SCALE_NONE;
    IT_CHECK_ARG(!scaled || (std::isfinite(c->factor) && c->factor >= 1.0), "it_rope_create: a scaling factor must be at least 1");
    IT_CHECK_ARG(c->scaling != IT_ROPE_SCALE_NTK || c->n_rot > 2, "it_rope_create: this scaling needs more than one pair");
    IT_CHECK_ARG(c->scaling != IT_ROPE_SCALE_YARN || (std::isfinite(c->original_ctx) && c->original_ctx >= 1.0 && std::isfinite(c->beta_fast) && c->beta_slow > 0.0 && c->beta_fast >= c->beta_slow),
                 "it_rope_create: the original context must be at least 1 and beta_fast >= beta_slow > 0");
    it_rope* r = new (std::nothrow) it_rope();
    if (!r) return it_fail(IT_ENOMEM, "it_rope_create: out of memory");
    r->n_rot = c->n_rot; r->layout = c->layout; r->mscale = 1.0;
    const int n = c->n_rot;
    const long double two_pi = 6.283185307179586476925286766559005768L;
    long double base = c->base;
    if (c->scaling == IT_ROPE_SCALE_NTK) base *= powl(c->factor, (long double)n / (n - 2));
    long double lo = 0, hi = 0;
    if (c->scaling == IT_ROPE_SCALE_YARN) {
        auto pair_of = [&](double turns) { return n * logl(c->original_ctx / (turns * two_pi)) / (2 * logl(base)); };   // the pair that turns so often in the original context
        lo = fmaxl(floorl(pair_of(c->beta_fast)), 0); hi = fminl(ceill(pair_of(c->beta_slow)), n - 1);
        r->mscale = 0.1 * std::log(c->factor) + 1.0;
    }
    for (int i = 0; i < n / 2; i++) {
        long double f = powl(base, -2.0L * i / n);
        if (c->scaling == IT_ROPE_SCALE_LINEAR) f /= c->factor;
        if (c->scaling == IT_ROPE_SCALE_YARN) {
            const long double s = fminl(fmaxl((i - lo) / fmaxl(hi - lo, 0.001L), 0), 1);
            f = f * (1 - s) + f / c->factor * s;
        }
        r->freq[i] = (double)f;
        r->turns[i] = (unsigned long long)roundl(f / two_pi * 18446744073709551616.0L);       // f <= 1 radian: below 2^62
    }
    *out = r;
    return IT_OK;
}
IT_API void it_rope_destroy(it_rope* r) { delete r; }
IT_API int it_rope_read(const it_rope* r, double* freq, double* mscale) {
    IT_CHECK_ARG(r, "it_rope_read: null argument");
    if (freq) for (int i = 0; i < r->n_rot / 2; i++) freq[i] = r->freq[i];
    if (mscale) *mscale = r->mscale;
    return IT_OK;
}

IT_API int it_norm_rope(void* stream, const it_norm_rope_args* a) {
    const char* const who = "it_norm_rope";
    IT_CHECK_ARG(a, "%s: null argument", who);
    IT_CHECK_ARG(it_type_pair(a->type, a->cache_type), "%s: types %d over %d", who, a->type, a->cache_type);
    IT_CHECK_ARG(a->rows >= 0 && a->rows <= (1 << 24), "%s: %d rows", who, a->rows);
    IT_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= NR_MAXDIM && a->head_dim % 8 == 0, "%s: head dimension %d is not a multiple of 8 up to 256", who, a->head_dim);
    IT_CHECK_ARG(a->kv_heads >= 1 && a->heads >= 1 && a->heads <= 65536 && a->heads % a->kv_heads == 0, "%s: %d heads over %d kv heads", who, a->heads, a->kv_heads);
    IT_CHECK_ARG(a->eps >= 0.f && a->eps <= 3e38f, "%s: bad eps", who);
    IT_CHECK_ARG(!a->rope || a->rope->n_rot <= a->head_dim, "%s: %d rotated elements in heads of %d", who, a->rope ? a->rope->n_rot : 0, a->head_dim);
    if (a->rows == 0) return IT_OK;
    IT_CHECK_ARG(a->q || a->k, "%s: neither q nor k", who);
    IT_CHECK_ARG(!a->k == !a->v, "%s: k and v come together", who);
    const size_t es = it_type_size(a->type), al = 4 * es;
    const int64_t T = a->rows, H = a->heads, G = a->kv_heads, D = a->head_dim;
    size_t qspan = 0, kspan = 0, vspan = 0;
    if (a->q) {
        IT_CHECK_ARG(a->q_out, "%s: q without q_out", who);
        IT_CHECK_ARG(it_aligned(a->q, al) && it_aligned(a->q_out, al) && it_strides_ok(T, a->q_row, H, a->q_head, D, 4) && it_strides_ok(T, a->qo_row, H, a->qo_head, D, 4),
                     "%s: q or q_out: pointers and strides are multiples of 4 elements, strides hold what lies between", who);
        qspan = it_span(T, a->q_row, H, a->q_head, D, es);
        const size_t os = it_span(T, a->qo_row, H, a->qo_head, D, es);
        const bool same = a->q == a->q_out && (T < 2 || a->q_row == a->qo_row) && (H < 2 || a->q_head == a->qo_head);
        IT_CHECK_ARG(same || !it_overlap(a->q, qspan, a->q_out, os), "%s: q_out overlaps q with another layout", who);
        if (a->k) {
            kspan = it_span(T, a->k_row, G, a->k_head, D, es); vspan = it_span(T, a->v_row, G, a->v_head, D, es);
            IT_CHECK_ARG(same || (!it_overlap(a->k, kspan, a->q_out, os) && !it_overlap(a->v, vspan, a->q_out, os)), "%s: q_out overlaps k or v", who);
        }
    }
    if (a->k) {
        IT_CHECK_ARG(a->k_cache && a->v_cache, "%s: k and v without caches", who);
        IT_CHECK_ARG(it_aligned(a->k, al) && it_aligned(a->v, al) && it_strides_ok(T, a->k_row, G, a->k_head, D, 4) && it_strides_ok(T, a->v_row, G, a->v_head, D, 4),
                     "%s: k or v: pointers and strides are multiples of 4 elements, strides hold what lies between", who);
        IT_CHECK_ARG(it_aligned(a->k_cache, 16) && it_aligned(a->v_cache, 16) && a->slots >= 1 && a->slots <= 0x7fffffffll && it_strides_ok(a->slots, a->kc_slot, G, a->kc_head, D, 8) &&
                     it_strides_ok(a->slots, a->vc_slot, G, a->vc_head, D, 8), "%s: caches: 16-byte aligned, strides are multiples of 8 elements and hold what lies between", who);
        const it_stretch caches[] = { { "k_cache", a->k_cache, it_span(a->slots, a->kc_slot, G, a->kc_head, D, 2) }, { "v_cache", a->v_cache, it_span(a->slots, a->vc_slot, G, a->vc_head, D, 2) } };
        if (const char* x = a->q ? it_overlaps({ "q_out", a->q_out, it_span(T, a->qo_row, H, a->qo_head, D, es) }, caches, 2) : nullptr) return it_fail(IT_EINVAL, "%s: q_out overlaps %s", who, x);
        IT_CHECK_ARG(a->slot0 >= 0 && a->slot0 <= a->slots && (a->base || a->slot0 + T <= a->slots), "%s: rows at slots %lld .. of %lld", who, (long long)a->slot0, (long long)a->slots);
    }
    IT_CHECK_ARG(it_aligned(a->positions, 4) && it_aligned(a->base, 4) && it_aligned(a->q_norm, 16) && it_aligned(a->k_norm, 16), "%s: a pointer is not aligned to its type (norm weights: 16 bytes)", who);
    it_ops_device dev;
    if (const int r = it_ops_current(stream, who, &dev)) return r;
    NrParams p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->q_out; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
    p.q_row = a->q_row; p.q_head = a->q_head; p.k_row = a->k_row; p.k_head = a->k_head; p.v_row = a->v_row; p.v_head = a->v_head; p.qo_row = a->qo_row; p.qo_head = a->qo_head;
    p.kc_slot = a->kc_slot; p.kc_head = a->kc_head; p.vc_slot = a->vc_slot; p.vc_head = a->vc_head; p.slots = a->slots; p.slot0 = a->slot0;
    p.positions = a->positions; p.base = a->base; p.q_norm = a->q_norm; p.k_norm = a->k_norm;
    p.rows = a->rows; p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->head_dim; p.pos0 = a->pos0; p.eps = a->eps;
    p.pairs = a->rope ? a->rope->n_rot / 2 : 0; p.interleaved = a->rope && a->rope->layout == IT_ROPE_INTERLEAVED; p.mscale = a->rope ? (float)a->rope->mscale : 1.f;
    for (int i = 0; i < p.pairs; i++) p.turns[i] = a->rope->turns[i];
    const int jobs = (a->q ? a->heads : 0) + (a->k ? 2 * a->kv_heads : 0);
    // A CTA has eight heads of a row; all of a row's where the rows alone fill the GPU, which makes its table once (24 + 4 + 4 heads, 4096 rows: 45.0 us; with eight heads a CTA 51.6, issue-bound).
    const unsigned groups = (unsigned)((jobs + NR_WARPS - 1) / NR_WARPS);
    const dim3 grid((unsigned)a->rows, a->rows >= 4 * dev.sm_count ? 1u : groups);
    const cudaStream_t st = (cudaStream_t)stream;
    const dim3 block(NR_WARPS * 32);
    if (a->type == IT_F32) IT_CUDA(it_launch_early(k_norm_rope<float, __half>, grid, block, 0, st, 1, p));
    else if (a->type == IT_F16) IT_CUDA(it_launch_early(k_norm_rope<__half, __half>, grid, block, 0, st, 1, p));
    else IT_CUDA(it_launch_early(k_norm_rope<__nv_bfloat16, __nv_bfloat16>, grid, block, 0, st, 1, p));
    return IT_OK;
}
