// kv_cache.cu -- step plans (request lengths to cache slots) and the 8-bit
// KV cache: quantising append and read-back.
#include "serving_common.cuh"

namespace hxq {
namespace serving {

// ---------------------------------------------------------------------------
// Step plan.
//   starts = exclusive sum of new, need[b] = ceil((c + n)/P) - ceil(c/P),
//   base = exclusive sum of need, entry ceil(c/P) + j of row b = free[base[b] + j],
//   slot of token i of b = entry[(c + i)/P] * P + (c + i) % P.
// A token in a block this step begins gets its entry from the free list
// itself, so no CTA reads what another one writes and one launch does it all:
// every CTA sums the lengths (8 bytes a request out of L2, a block scan) and
// then fills its own part of the slot map and of the table.  Bound by the
// launch and two dependent loads, not by bytes.

constexpr int kPlanThreads = 512;

struct PlanArgs {
    const int32_t *n, *c, *free_list;
    int32_t *table, *starts, *lens, *slots, *positions, *taken;
    uint32_t *status;
    uint32_t B, width, P, n_free, n_slots;
};

__device__ __forceinline__ uint32_t last_at_most(const uint32_t *v, uint32_t n, uint32_t x)
{
    // the last i < n with v[i] <= x (v ascending, v[0] = 0)
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a)
{
    extern __shared__ uint32_t sm[];
    uint32_t *starts = sm, *base = sm + a.B + 1;
    __shared__ unsigned long long wsum[2][kPlanThreads / 32];
    __shared__ unsigned long long carry[2];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr uint64_t kMost = 0x7fffffffull;
    if (tid < 2) carry[tid] = 0;
    __syncthreads();
    uint32_t bad = 0;
    for (uint32_t b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint64_t n = 0, need = 0;
        if (b < a.B) {
            int32_t ni = a.n[b], ci = a.c[b];
            if (ni < 0 || ci < 0) bad |= HXQ_SERVING_BAD_LENGTH;
            n = ni < 0 ? 0 : ni;
            const uint64_t c = ci < 0 ? 0 : ci;
            uint64_t len = c + n;
            if (len > kMost) bad |= HXQ_SERVING_BAD_LENGTH;
            need = (len + a.P - 1) / a.P - (c + a.P - 1) / a.P;
            if (blockIdx.x == 0) a.lens[b] = (int32_t)(len > kMost ? kMost : len);
        }
        unsigned long long x = n, y = need;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned long long u = __shfl_up_sync(~0u, x, d), v = __shfl_up_sync(~0u, y, d);
            if (lane >= d) { x += u; y += v; }
        }
        if (lane == 31) { wsum[0][warp] = x; wsum[1][warp] = y; }
        __syncthreads();
        unsigned long long px = carry[0], py = carry[1];
        for (uint32_t w = 0; w < warp; ++w) { px += wsum[0][w]; py += wsum[1][w]; }
        x += px;
        y += py;
        if (b < a.B) {
            const uint64_t s = x - n, e = y - need;
            starts[b] = (uint32_t)(s < kMost ? s : kMost);
            base[b] = (uint32_t)(e < kMost ? e : kMost);
        }
        __syncthreads();
        if (tid == kPlanThreads - 1) { carry[0] = x; carry[1] = y; }
        __syncthreads();
    }
    const uint32_t total = (uint32_t)(carry[0] < kMost ? carry[0] : kMost);
    const uint32_t fresh = (uint32_t)(carry[1] < kMost ? carry[1] : kMost);
    if (tid == 0) { starts[a.B] = total; base[a.B] = fresh; }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (uint32_t b = tid; b <= a.B; b += kPlanThreads) a.starts[b] = (int32_t)starts[b];
        if (tid == 0) {
            a.taken[0] = (int32_t)min(fresh, a.n_free);
            if (fresh > a.n_free) bad |= HXQ_SERVING_NO_BLOCKS;
            if (total > a.n_slots) bad |= HXQ_SERVING_FULL;
        }
    }
    const uint32_t first = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
    // entries of the blocks this step begins
    for (uint32_t e = first; e < fresh; e += step) {
        const uint32_t b = last_at_most(base, a.B, e);
        const uint32_t c = (uint32_t)max(a.c[b], 0);
        const uint64_t at = (c + (uint64_t)a.P - 1) / a.P + (e - base[b]);
        if (at < a.width) a.table[(size_t)b * a.width + at] = e < a.n_free ? a.free_list[e] : -1;
        else bad |= HXQ_SERVING_BAD_BLOCK;
    }
    for (uint32_t t = first; t < a.n_slots; t += step) {
        int32_t slot = -1, pos = -1;
        if (t < total) {
            const uint32_t b = last_at_most(starts, a.B, t);
            const uint32_t c = (uint32_t)max(a.c[b], 0);
            const uint64_t p = (uint64_t)c + (t - starts[b]);
            const uint32_t held = (c + a.P - 1) / a.P;
            const uint64_t blk = p / a.P;
            int32_t block = -1;
            if (blk >= a.width) bad |= HXQ_SERVING_BAD_BLOCK;
            else if (blk < held) block = a.table[(size_t)b * a.width + blk];
            else {
                const uint64_t e = base[b] + (blk - held);
                block = e < a.n_free ? a.free_list[e] : -1;
                if (e < a.n_free && block < 0) bad |= HXQ_SERVING_BAD_BLOCK;
            }
            if (blk < held && block < 0) bad |= HXQ_SERVING_BAD_BLOCK;
            pos = (int32_t)(p > kMost ? kMost : p);
            const int64_t s = (int64_t)block * a.P + (int64_t)(p % a.P);
            if (block >= 0 && s <= (int64_t)kMost) slot = (int32_t)s;
            else if (block >= 0) bad |= HXQ_SERVING_BAD_BLOCK;
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    if (bad) flag(a.status, bad);
}

// ---------------------------------------------------------------------------
// Append.  The unit of work is one (run, head, k or v): a run is the rows of
// one block that follow each other in the call.  A warp finds the largest
// magnitude of the run, merges it with the block's scale, writes the run's
// codes and, when the scale grew, rounds the block's other codes to the new
// one.  Bound by the bytes of the rows (the second look at a run hits L1/L2).
//
// Magnitudes are compared as the integers of their bits (non-negative floats
// order like integers, NaN above all), so infinities and NaN reach the scale.
// x * (1/s') instead of x / s': one division for a block instead of one per
// value; the code differs from the quotient's by a tie within 1.5 ulp.
// Code and value of a block whose scale did not change stay as they are.

constexpr int kAppendWarps = 8;

struct AppendArgs {
    const void *x[2];
    uint8_t *codes[2];
    float *scales[2];
    int64_t st[2], sh[2];
    const int32_t *slots;
    uint32_t *status;
    uint32_t n_tokens, n_heads, P, D, n_blocks, window;
};

template <typename T, int VEC> struct Pack { T v[VEC]; };

template <typename T, int VEC> __device__ __forceinline__ void load_row(float (&f)[8], const T *p)
{
    if (VEC == 8) {
        constexpr int W = sizeof(T) * 8 / 16;
        uint4 raw[W];
#pragma unroll
        for (int i = 0; i < W; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to(p[i]);
    }
}

template <int FMT> __device__ __forceinline__ uint2 pack_codes(const float (&f)[8], float m)
{
    uint2 r;
    if (FMT == HXQ_KV_INT8) {
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t a = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) a |= (uint32_t)nearest_code<FMT>(f[4 * h + i] * m) << (8 * i);
            w[h] = a;
        }
        r.x = w[0];
        r.y = w[1];
    } else {
        uint16_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * m, f[2 * i + 1] * m), __NV_SATFINITE, __NV_E4M3);
        r.x = q[0] | (uint32_t)q[1] << 16;
        r.y = q[2] | (uint32_t)q[3] << 16;
    }
    return r;
}

template <typename T, int FMT, int VEC>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(const AppendArgs a)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t item = blockIdx.y * kAppendWarps + warp;   // (head, k or v)
    if (item >= a.n_heads * 2) return;
    const uint32_t kv = item & 1, h = item >> 1;
    const T *x = static_cast<const T *>(a.x[kv]) + (int64_t)h * a.sh[kv];
    const int64_t st = a.st[kv];
    const uint32_t n_slots = a.n_blocks * a.P, lg = a.D == 64 ? 3 : a.D == 128 ? 4 : 5;   // 8-value pieces a row
    const float qmax = FMT == HXQ_KV_INT8 ? 127.0f : 448.0f;
    const uint32_t t_begin = blockIdx.x * a.window, t_end = min(t_begin + a.window, a.n_tokens);
    for (uint32_t t0 = t_begin; t0 < t_end; t0 += 32) {
        // which rows of the window begin a run
        const uint32_t tl = t0 + lane;
        bool lead = false;
        if (tl < t_end) {
            const int32_t s = a.slots[tl], before = tl ? a.slots[tl - 1] : -1;
            if (s >= 0) {
                if ((uint32_t)s >= n_slots) {
                    if (item == 0) flag(a.status, HXQ_SERVING_BAD_BLOCK);
                } else {
                    const bool same = before >= 0 && (uint32_t)before / a.P == (uint32_t)s / a.P;
                    lead = !same || before >= s;
                    if (same && before >= s && item == 0) flag(a.status, HXQ_SERVING_ORDER);
                }
            }
        }
        uint32_t leads = __ballot_sync(~0u, lead);
        while (leads) {
            const uint32_t t = t0 + __ffs(leads) - 1;
            leads &= leads - 1;
            const uint32_t s0 = (uint32_t)a.slots[t], block = s0 / a.P, pos0 = s0 % a.P;
            // length of the run (at most P rows) and the block's positions it writes
            uint32_t len = 0, mine[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            for (bool more = true; more;) {
                const uint32_t u = t + len + lane;
                bool in = u < a.n_tokens;
                uint32_t p = 0;
                if (in) {
                    const int32_t s = a.slots[u];
                    in = s >= 0 && (uint32_t)s / a.P == block && (u == t || s > a.slots[u - 1]);
                    p = (uint32_t)s % a.P;
                }
                const uint32_t yes = __ballot_sync(~0u, in), n = yes == ~0u ? 32u : (uint32_t)__ffs(~yes) - 1;
                if (lane >= n) in = false;
#pragma unroll
                for (int w = 0; w < 8; ++w)
                    mine[w] |= __reduce_or_sync(~0u, in && (p >> 5) == (uint32_t)w ? 1u << (p & 31) : 0u);
                len += n;
                more = n == 32;
            }
            // largest magnitude of the run
            const uint32_t pieces = len << lg;
            uint32_t top = 0;
#pragma unroll 4
            for (uint32_t e = lane; e < pieces; e += 32) {
                float f[8];
                load_row<T, VEC>(f, x + (int64_t)(t + (e >> lg)) * st + (e & ((1u << lg) - 1)) * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
            }
            top = __reduce_max_sync(~0u, top);
            float *scale_at = a.scales[kv] + (size_t)block * a.n_heads + h;
            const float old = pos0 == 0 ? 0.0f : *scale_at;
            float scale = __uint_as_float(max(__float_as_uint(old) & 0x7fffffffu, __float_as_uint(__uint_as_float(top) / qmax)));
            if (scale < 1.17549435e-38f) scale = 0.0f;
            const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
            const bool lost = !(scale <= 3.402823466e38f);   // infinite or NaN: the codes are 0, so that no code is NaN
            uint8_t *codes = a.codes[kv] + ((size_t)block * a.n_heads + h) * a.P * a.D;
            const bool grew = pos0 != 0 && !(scale <= old);
            __syncwarp();
            if (lane == 0) *scale_at = scale;
#pragma unroll 4
            for (uint32_t e = lane; e < pieces; e += 32) {
                const uint32_t u = t + (e >> lg), col = (e & ((1u << lg) - 1)) * 8;
                float f[8];
                load_row<T, VEC>(f, x + (int64_t)u * st + col);
                *reinterpret_cast<uint2 *>(codes + (size_t)((uint32_t)a.slots[u] % a.P) * a.D + col) =
                    lost ? make_uint2(0u, 0u) : pack_codes<FMT>(f, inv);
            }
            if (grew) {
                const float ratio = scale > 0.0f ? old / scale : 0.0f;
                for (uint32_t e = lane; e < a.P << lg; e += 32) {
                    const uint32_t p = e >> lg;
                    uint32_t word = 0;
#pragma unroll
                    for (int w = 0; w < 8; ++w) word = (p >> 5) == (uint32_t)w ? mine[w] : word;
                    if (word >> (p & 31) & 1u) continue;
                    uint2 *at = reinterpret_cast<uint2 *>(codes + (size_t)e * 8);
                    const uint2 was = *at;
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = code_value<FMT>((uint8_t)((i < 4 ? was.x : was.y) >> (8 * (i & 3))));
                    *at = pack_codes<FMT>(f, ratio);
                }
            }
        }
    }
}

// Read-back: one thread per 8 values of k and of v.
template <typename T, int FMT>
__global__ void read_kernel(const hxq_kv_cache_t c, const int32_t *slots, uint32_t n_tokens, T *k, T *v, uint32_t *status)
{
    const uint32_t lg = c.head_dim == 64 ? 3 : c.head_dim == 128 ? 4 : 5, per = c.n_heads << lg;
    const uint64_t n = (uint64_t)n_tokens * per, step = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const uint32_t t = (uint32_t)(i / per), r = (uint32_t)(i - (uint64_t)t * per), h = r >> lg, col = (r & ((1u << lg) - 1)) * 8;
        const int32_t s = slots[t];
        const bool ok = s >= 0 && (uint32_t)s < c.n_blocks * c.block_tokens;
        if (s >= 0 && !ok && r == 0) flag(status, HXQ_SERVING_BAD_BLOCK);
        const uint32_t block = ok ? (uint32_t)s / c.block_tokens : 0, pos = ok ? (uint32_t)s % c.block_tokens : 0;
        const size_t bh = (size_t)block * c.n_heads + h, at = (bh * c.block_tokens + pos) * c.head_dim + col;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            T *out = w ? v : k;
            if (!out) continue;
            T o[8];
            if (ok) {
                const uint2 raw = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(w ? c.v : c.k) + at));
                const float scale = (w ? c.v_scales : c.k_scales)[bh];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    o[j] = Elem<T>::from(code_value<FMT>((uint8_t)((j < 4 ? raw.x : raw.y) >> (8 * (j & 3)))) * scale);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = Elem<T>::from(0.0f);
            }
            T *dst = out + ((size_t)t * c.n_heads + h) * c.head_dim + col;
            if ((((uintptr_t)out) & 15u) == 0) {
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                    reinterpret_cast<uint4 *>(dst)[j] = reinterpret_cast<const uint4 *>(o)[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[j] = o[j];
            }
        }
    }
}

template <typename T, int FMT> void launch_append(const AppendArgs &a, bool vec, dim3 grid, cudaStream_t s)
{
    if (vec) append_kernel<T, FMT, 8><<<grid, kAppendWarps * 32, 0, s>>>(a);
    else append_kernel<T, FMT, 1><<<grid, kAppendWarps * 32, 0, s>>>(a);
}

}  // namespace serving
}  // namespace hxq

using namespace hxq::serving;

extern "C" {

hxq_error_t hxq_cuda_kv_plan(const int32_t *d_new, const int32_t *d_cached, uint32_t B, int32_t *d_table,
                             uint32_t table_width, uint32_t block_tokens, const int32_t *d_free, uint32_t n_free,
                             int32_t *d_starts, int32_t *d_lens, int32_t *d_slots, int32_t *d_positions,
                             uint32_t n_slots, int32_t *d_taken, uint32_t *d_status, void *stream)
{
    if (!d_starts || !d_taken || (B && (!d_new || !d_cached || !d_lens || (!d_table && table_width))) || (n_free && !d_free) ||
        (n_slots && (!d_slots || !d_positions)))
        return HXQ_ERR_NULL_PTR;
    if (B > HXQ_PLAN_MAX_REQUESTS || block_tokens == 0 || block_tokens > 65536u || n_slots > 0x7fffffffu ||
        n_free > 0x7fffffffu)
        return HXQ_ERR_INVALID_ARG;
    PlanArgs a = {d_new, d_cached, d_free, d_table, d_starts, d_lens, d_slots, d_positions, d_taken, d_status,
                  B, table_width, block_tokens, n_free, n_slots};
    const size_t smem = (size_t)(B + 1) * 2 * sizeof(uint32_t);
    static std::atomic<uint64_t> ready{0};
    if (smem > 48u * 1024u &&
        allow_smem(plan_kernel, (HXQ_PLAN_MAX_REQUESTS + 1) * 2 * sizeof(uint32_t), ready) != cudaSuccess) {
        cudaGetLastError();
        return HXQ_ERR_CUDA;
    }
    const uint32_t want = (n_slots + kPlanThreads - 1) / kPlanThreads, most = 2u * (uint32_t)sm_count();
    const uint32_t grid = want == 0 ? 1 : want < most ? want : most;
    plan_kernel<<<grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    return launched();
}

hxq_error_t hxq_cuda_kv_append(const hxq_kv_cache_t *cache, const void *d_k, const void *d_v, int elem,
                               int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                               const int32_t *d_slots, uint32_t n_tokens, uint32_t *d_status, void *stream)
{
    const hxq_error_t err = check_cache(cache);
    if (err != HXQ_OK) return err;
    if (elem != HXQ_ELEM_F32 && elem != HXQ_ELEM_BF16 && elem != HXQ_ELEM_F16) return HXQ_ERR_INVALID_ARG;
    if (n_tokens > 0x7fffffffu) return HXQ_ERR_INVALID_ARG;
    if (n_tokens == 0) return HXQ_OK;
    if (!d_k || !d_v || !d_slots) return HXQ_ERR_NULL_PTR;
    const uintptr_t size = elem == HXQ_ELEM_F32 ? 4 : 2;
    if (((uintptr_t)d_k | (uintptr_t)d_v) & (size - 1)) return HXQ_ERR_INVALID_ARG;
    AppendArgs a;
    a.x[0] = d_k;
    a.x[1] = d_v;
    a.codes[0] = static_cast<uint8_t *>(cache->k);
    a.codes[1] = static_cast<uint8_t *>(cache->v);
    a.scales[0] = cache->k_scales;
    a.scales[1] = cache->v_scales;
    a.st[0] = k_stride_t;
    a.st[1] = v_stride_t;
    a.sh[0] = k_stride_h;
    a.sh[1] = v_stride_h;
    a.slots = d_slots;
    a.status = d_status;
    a.n_tokens = n_tokens;
    a.n_heads = cache->n_heads;
    a.P = cache->block_tokens;
    a.D = cache->head_dim;
    a.n_blocks = cache->n_blocks;
    // rows a CTA looks for runs in: one when there are few (each run a warp of
    // its own), up to 64 when there are enough to fill the GPU all the same
    const uint64_t fill = (uint64_t)n_tokens * cache->n_heads * 2 / ((uint64_t)sm_count() * 32);
    a.window = (uint32_t)(fill < 1 ? 1 : fill > 64 ? 64 : fill);
    const dim3 grid((n_tokens + a.window - 1) / a.window, (cache->n_heads * 2 + kAppendWarps - 1) / kAppendWarps);
    // 16-byte loads where every row begins on a 16-byte boundary
    const uint64_t s = (uint64_t)(k_stride_t | k_stride_h | v_stride_t | v_stride_h) * size;
    const bool vec = ((s | (uintptr_t)d_k | (uintptr_t)d_v) & 15u) == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool i8 = cache->format == HXQ_KV_INT8;
    if (elem == HXQ_ELEM_F32) i8 ? launch_append<float, HXQ_KV_INT8>(a, vec, grid, st) : launch_append<float, HXQ_KV_E4M3>(a, vec, grid, st);
    else if (elem == HXQ_ELEM_BF16)
        i8 ? launch_append<__nv_bfloat16, HXQ_KV_INT8>(a, vec, grid, st) : launch_append<__nv_bfloat16, HXQ_KV_E4M3>(a, vec, grid, st);
    else i8 ? launch_append<__half, HXQ_KV_INT8>(a, vec, grid, st) : launch_append<__half, HXQ_KV_E4M3>(a, vec, grid, st);
    return launched();
}

hxq_error_t hxq_cuda_kv_read(const hxq_kv_cache_t *cache, const int32_t *d_slots, uint32_t n_tokens, void *d_k,
                             void *d_v, int elem, uint32_t *d_status, void *stream)
{
    const hxq_error_t err = check_cache(cache);
    if (err != HXQ_OK) return err;
    if (elem != HXQ_ELEM_F32 && elem != HXQ_ELEM_BF16 && elem != HXQ_ELEM_F16) return HXQ_ERR_INVALID_ARG;
    if (n_tokens > 0x7fffffffu) return HXQ_ERR_INVALID_ARG;
    if (n_tokens == 0) return HXQ_OK;
    if (!d_slots || (!d_k && !d_v)) return HXQ_ERR_NULL_PTR;
    const uintptr_t size = elem == HXQ_ELEM_F32 ? 4 : 2;
    if (((uintptr_t)d_k | (uintptr_t)d_v) & (size - 1)) return HXQ_ERR_INVALID_ARG;
    const uint64_t n = (uint64_t)n_tokens * cache->n_heads * (cache->head_dim / 8), want = (n + 255) / 256;
    const uint64_t most = (uint64_t)sm_count() * 16;
    const unsigned grid = (unsigned)(want < most ? want : most);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool i8 = cache->format == HXQ_KV_INT8;
#define HXQ_READ(T)                                                                                                  \
    (i8 ? read_kernel<T, HXQ_KV_INT8><<<grid, 256, 0, s>>>(*cache, d_slots, n_tokens, (T *)d_k, (T *)d_v, d_status)   \
        : read_kernel<T, HXQ_KV_E4M3><<<grid, 256, 0, s>>>(*cache, d_slots, n_tokens, (T *)d_k, (T *)d_v, d_status))
    if (elem == HXQ_ELEM_F32) HXQ_READ(float);
    else if (elem == HXQ_ELEM_BF16) HXQ_READ(__nv_bfloat16);
    else HXQ_READ(__half);
#undef HXQ_READ
    return launched();
}

}  // extern "C"
