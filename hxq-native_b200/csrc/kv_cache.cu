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
// launch and two dependent loads, not by bytes: 8.5 us a call for 64 decoding
// requests and for 500 prompts of up to 1024 tokens.

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
// one block that follow each other in the call.  G warps find the largest
// magnitude of the run, merge it with the block's scale, write the run's codes
// and, when the scale grew, round the block's other codes to the new one.  A
// lane keeps up to 8 pieces of 8 values between the two looks at a run, G
// chosen so that a whole block's rows fit (blocks beyond 8 warps' worth are
// read again, out of L2).  Bound by the latency of a run (slots, then rows,
// then codes, with no more warps an SM than the held pieces' registers allow;
// fewer registers spill and cost more; half the pieces with twice the
// warps a run: 140 us for both kernels): 77 us for 9 prompts of up to 2048 rows,
// 32 heads of 128, bf16 to e4m3, where the bytes take 36.  Rows read
// twice instead of held: 149 us with the read-back against 130, 128 with the next
// run's rows brought to L2 while this one's are looked at.
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

template <typename T> struct Piece {   // 8 values as they are in memory
    static constexpr int kWords = sizeof(T) * 8 / 16;
    uint4 raw[kWords];
};

// 16-byte loads where VEC, else one by one.
template <typename T, bool VEC> __device__ __forceinline__ Piece<T> load_piece(const T *p)
{
    Piece<T> v;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < Piece<T>::kWords; ++i) v.raw[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::kWords; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (sizeof(T) == 4) w[u] = reinterpret_cast<const uint32_t *>(p)[i * 4 + u];
                else {
                    const uint16_t *e = reinterpret_cast<const uint16_t *>(p) + 2 * u;
                    w[u] = e[0] | (uint32_t)e[1] << 16;
                }
            }
            v.raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    return v;
}

__device__ __forceinline__ float2 pair_of(uint32_t w, const float *) { return make_float2(__uint_as_float(w), 0.0f); }
__device__ __forceinline__ float2 pair_of(uint32_t w, const __nv_bfloat16 *)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, const __half *)
{
    return __half22float2(__halves2half2(__ushort_as_half((uint16_t)w), __ushort_as_half((uint16_t)(w >> 16))));
}

template <typename T> __device__ __forceinline__ void values(const Piece<T> &v, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < Piece<T>::kWords; ++i) {
        const uint32_t w[4] = {v.raw[i].x, v.raw[i].y, v.raw[i].z, v.raw[i].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float2 p = pair_of(w[u], static_cast<const T *>(nullptr));
            if (sizeof(T) == 4) f[(i * 4 + u) & 7] = p.x;
            else {
                f[(2 * u) & 7] = p.x;
                f[(2 * u + 1) & 7] = p.y;
            }
        }
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

constexpr int kHeld = 8;   // pieces a lane keeps

template <typename T, int FMT, bool VEC, int G>
__global__ void __launch_bounds__(kAppendWarps * 32, sizeof(T) == 4 ? 2 : 3) append_kernel(const AppendArgs a)
{
    __shared__ uint32_t tops[2][kAppendWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wg = warp % G;
    // CTAs of the same rows follow each other, so that whole rows of the call
    // are under way at once
    const uint32_t groups = (a.n_heads * 2 + kAppendWarps / G - 1) / (kAppendWarps / G), window = blockIdx.x / groups;
    const uint32_t item = (blockIdx.x - window * groups) * (kAppendWarps / G) + warp / G;   // (head, k or v)
    const bool mine_too = item < a.n_heads * 2;                         // the CTA's warps stay together
    const uint32_t kv = item & 1, h = mine_too ? item >> 1 : 0;
    const T *x = static_cast<const T *>(kv ? a.x[1] : a.x[0]) + (int64_t)h * (kv ? a.sh[1] : a.sh[0]);
    const int64_t st = kv ? a.st[1] : a.st[0];
    const uint32_t n_slots = a.n_blocks * a.P, lg = a.D == 64 ? 3 : a.D == 128 ? 4 : 5;   // 8-value pieces a row
    const float qmax = FMT == HXQ_KV_INT8 ? 127.0f : 448.0f;
    const uint32_t t_begin = window * a.window, t_end = min(t_begin + a.window, a.n_tokens);
    uint32_t turn = 0;
    for (uint32_t t0 = t_begin; t0 < t_end; t0 += 32) {
        // which rows of the window begin a run
        const uint32_t tl = t0 + lane;
        bool lead = false;
        if (tl < t_end) {
            const int32_t s = a.slots[tl], before = tl ? a.slots[tl - 1] : -1;
            if (s >= 0) {
                if ((uint32_t)s >= n_slots) {
                    if (item == 0 && wg == 0) flag(a.status, HXQ_SERVING_BAD_BLOCK);
                } else {
                    const bool same = before >= 0 && (uint32_t)before / a.P == (uint32_t)s / a.P;
                    lead = !same || before >= s;
                    if (same && before >= s && item == 0 && wg == 0) flag(a.status, HXQ_SERVING_ORDER);
                }
            }
        }
        uint32_t leads = __ballot_sync(~0u, lead);
        while (leads) {
            const uint32_t t = t0 + __ffs(leads) - 1;
            leads &= leads - 1;
            const uint32_t s0 = (uint32_t)a.slots[t], block = s0 / a.P, pos0 = s0 - block * a.P;
            float *scale_at = (kv ? a.scales[1] : a.scales[0]) + (size_t)block * a.n_heads + h;
            const float old = pos0 == 0 ? 0.0f : *scale_at;
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
                if (pos0 != 0) {   // needed where codes are rounded again
#pragma unroll
                    for (int w = 0; w < 8; ++w)
                        mine[w] |= __reduce_or_sync(~0u, in && (p >> 5) == (uint32_t)w ? 1u << (p & 31) : 0u);
                }
                len += n;
                more = n == 32;
            }
            // largest magnitude of the run
            const uint32_t pieces = len << lg, e0 = wg * 32 + lane;
            auto row_at = [&](uint32_t e) { return x + (int64_t)(t + (e >> lg)) * st + (e & ((1u << lg) - 1)) * 8; };
            Piece<T> held[kHeld];
            uint32_t top = 0;
            auto look = [&](const Piece<T> &v) {
                float f[8];
                values(v, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
            };
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (e0 + i * (32 * G) < pieces) held[i] = load_piece<T, VEC>(row_at(e0 + i * (32 * G)));
            // the rows behind them on their way to L2 meanwhile
            {
                constexpr uint32_t kLine = 128 / sizeof(T);
                const uint32_t per = a.D / kLine, lgl = per == 1 ? 0 : per == 2 ? 1 : per == 4 ? 2 : 3;
                for (uint32_t e = e0; e < a.P << lgl; e += 32 * G) {
                    const uint32_t u = t + len + (e >> lgl);
                    if (u < t_end) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + (int64_t)u * st + (e & (per - 1)) * kLine));
                }
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (e0 + i * (32 * G) < pieces) look(held[i]);
            for (uint32_t e = e0 + kHeld * (32 * G); e < pieces; e += 32 * G) look(load_piece<T, VEC>(row_at(e)));
            top = __reduce_max_sync(~0u, top);
            if (G > 1) {
                if (lane == 0) tops[turn][warp] = top;
                __syncthreads();   // a lead is every warp's of the CTA: the slots are the same
#pragma unroll
                for (int w = 0; w < G; ++w) top = max(top, tops[turn][warp - wg + w]);
                turn ^= 1u;
            }
            float scale = __uint_as_float(max(__float_as_uint(old) & 0x7fffffffu, __float_as_uint(__uint_as_float(top) / qmax)));
            if (scale < 1.17549435e-38f) scale = 0.0f;
            const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
            const bool lost = !(scale <= 3.402823466e38f);   // infinite or NaN: the codes are 0, so that no code is NaN
            uint8_t *codes = (kv ? a.codes[1] : a.codes[0]) + ((size_t)block * a.n_heads + h) * a.P * a.D;
            const bool grew = pos0 != 0 && !(scale <= old);
            if (!mine_too) continue;
            const bool dense = (uint32_t)a.slots[t + len - 1] - s0 == len - 1;   // ascending: no gaps
            auto put = [&](uint32_t e, const Piece<T> &v) {
                float f[8];
                values(v, f);
                const uint32_t at = dense ? pos0 + (e >> lg) : (uint32_t)a.slots[t + (e >> lg)] - block * a.P;
                *reinterpret_cast<uint2 *>(codes + (size_t)at * a.D + (e & ((1u << lg) - 1)) * 8) =
                    lost ? make_uint2(0u, 0u) : pack_codes<FMT>(f, inv);
            };
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (e0 + i * (32 * G) < pieces) put(e0 + i * (32 * G), held[i]);
            for (uint32_t e = e0 + kHeld * (32 * G); e < pieces; e += 32 * G) put(e, load_piece<T, VEC>(row_at(e)));
            __syncwarp();   // (G > 1: the barrier above) the old scale is read
            if (lane == 0 && wg == 0) *scale_at = scale;
            if (grew) {
                const float ratio = scale > 0.0f ? old / scale : 0.0f;
                for (uint32_t e = e0; e < a.P << lg; e += 32 * G) {
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

// Read-back: a thread takes 16 consecutive codes of k or v, a CTA whole
// tokens, four of a thread's pieces under way.  Bound by memory: 48 us for the
// rows of the append above (e4m3 to bf16), where the bytes take 36.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) read_kernel(const hxq_kv_cache_t c, const int32_t *slots, uint32_t n_tokens, T *k, T *v, uint32_t *status)
{
    const uint32_t lg = c.head_dim == 64 ? 2 : c.head_dim == 128 ? 3 : 4, per = c.n_heads << lg;   // pieces of a token
    const uint32_t side = per < 256 ? 256 / per : 1, mine = threadIdx.x / per;                      // tokens side by side
    T *out = blockIdx.y ? v : k;
    if (!out || (per < 256 && mine >= side)) return;
    const uint8_t *codes = static_cast<const uint8_t *>(blockIdx.y ? c.v : c.k);
    const float *scales = blockIdx.y ? c.v_scales : c.k_scales;
    const uint32_t n_slots = c.n_blocks * c.block_tokens, step = gridDim.x * side;
    const bool wide = ((uintptr_t)out & 15u) == 0;
    for (uint32_t r = per < 256 ? threadIdx.x - mine * per : threadIdx.x; r < per; r += 256) {
        const uint32_t h = r >> lg, col = (r & ((1u << lg) - 1)) * 16;
        for (uint64_t t0 = (uint64_t)blockIdx.x * side + (per < 256 ? mine : 0); t0 < n_tokens; t0 += 4ull * step) {
            uint4 raw[4];
            float scale[4];
            bool ok[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint64_t t = t0 + (uint64_t)u * step;
                const int32_t s = t < n_tokens ? __ldg(slots + t) : -1;
                ok[u] = s >= 0 && (uint32_t)s < n_slots;
                if (s >= 0 && !ok[u] && r == 0) flag(status, HXQ_SERVING_BAD_BLOCK);
                const uint32_t block = ok[u] ? (uint32_t)s / c.block_tokens : 0, pos = ok[u] ? (uint32_t)s - block * c.block_tokens : 0;
                const size_t bh = (size_t)block * c.n_heads + h;
                raw[u] = make_uint4(0, 0, 0, 0);
                scale[u] = 0.0f;
                if (ok[u]) {
                    raw[u] = __ldg(reinterpret_cast<const uint4 *>(codes + (bh * c.block_tokens + pos) * c.head_dim + col));
                    scale[u] = __ldg(scales + bh);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint64_t t = t0 + (uint64_t)u * step;
                if (t >= n_tokens) break;
                const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                __align__(16) T o[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    o[j] = Elem<T>::from(ok[u] ? code_value<FMT>((uint8_t)(w[j >> 2] >> (8 * (j & 3)))) * scale[u] : 0.0f);
                T *dst = out + (t * c.n_heads + h) * c.head_dim + col;
                if (wide) {
#pragma unroll
                    for (int j = 0; j < (int)sizeof(T); ++j) reinterpret_cast<uint4 *>(dst)[j] = reinterpret_cast<const uint4 *>(o)[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) dst[j] = o[j];
                }
            }
        }
    }
}

// Warps of a run: a block's rows in kHeld pieces a lane.
template <typename T, int FMT> void launch_append(const AppendArgs &a, bool vec, uint32_t windows, cudaStream_t s)
{
    const uint32_t need = a.P * a.D / (8 * 32 * kHeld), g = !vec || need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
    const uint32_t grid = windows * ((a.n_heads * 2 + kAppendWarps / g - 1) / (kAppendWarps / g));
    constexpr int N = kAppendWarps * 32;
    if (!vec) append_kernel<T, FMT, false, 1><<<grid, N, 0, s>>>(a);
    else if (g == 1) append_kernel<T, FMT, true, 1><<<grid, N, 0, s>>>(a);
    else if (g == 2) append_kernel<T, FMT, true, 2><<<grid, N, 0, s>>>(a);
    else if (g == 4) append_kernel<T, FMT, true, 4><<<grid, N, 0, s>>>(a);
    else append_kernel<T, FMT, true, 8><<<grid, N, 0, s>>>(a);
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
    // CTAs read the lengths, the free list and the table while others write
    const struct { const void *at; uint64_t words; } parts[] = {
        {d_starts, (uint64_t)B + 1}, {d_lens, B}, {d_slots, n_slots}, {d_positions, n_slots}, {d_taken, 1},   // written
        {d_table, (uint64_t)B * table_width}, {d_new, B}, {d_cached, B}, {d_free, n_free}};
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 9; ++j) {
            const uint64_t x = (uint64_t)(uintptr_t)parts[i].at, y = (uint64_t)(uintptr_t)parts[j].at;
            if (parts[i].words && parts[j].words && x < y + 4 * parts[j].words && y < x + 4 * parts[i].words) return HXQ_ERR_INVALID_ARG;
        }
    PlanArgs a = {d_new, d_cached, d_free, d_table, d_starts, d_lens, d_slots, d_positions, d_taken, d_status,
                  B, table_width, block_tokens, n_free, n_slots};
    const size_t smem = (size_t)(B + 1) * 2 * sizeof(uint32_t);
    static std::atomic<uint64_t> ready{0};
    if (smem > 40u * 1024u &&   // 48 KB with the kernel's static part need no permission
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
    const uint32_t windows = (n_tokens + a.window - 1) / a.window;
    if ((uint64_t)windows * cache->n_heads * 2 > 0x7fffffffu) return HXQ_ERR_INVALID_ARG;
    // 16-byte loads where every row begins on a 16-byte boundary
    const uint64_t s = (uint64_t)(k_stride_t | k_stride_h | v_stride_t | v_stride_h) * size;
    const bool vec = ((s | (uintptr_t)d_k | (uintptr_t)d_v) & 15u) == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool i8 = cache->format == HXQ_KV_INT8;
    if (elem == HXQ_ELEM_F32) i8 ? launch_append<float, HXQ_KV_INT8>(a, vec, windows, st) : launch_append<float, HXQ_KV_E4M3>(a, vec, windows, st);
    else if (elem == HXQ_ELEM_BF16)
        i8 ? launch_append<__nv_bfloat16, HXQ_KV_INT8>(a, vec, windows, st) : launch_append<__nv_bfloat16, HXQ_KV_E4M3>(a, vec, windows, st);
    else i8 ? launch_append<__half, HXQ_KV_INT8>(a, vec, windows, st) : launch_append<__half, HXQ_KV_E4M3>(a, vec, windows, st);
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
    const uint32_t per = cache->n_heads * (cache->head_dim / 16), side = per < 256 ? 256 / per : 1;
    const uint32_t want = (n_tokens + side - 1) / side, most = (uint32_t)sm_count() * 4;
    const dim3 grid(want < most ? want : most, 2);
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
