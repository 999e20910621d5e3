// lora.cu -- low-rank adapters of many requests beside a shared projection:
//     out = y + s_a (x A_a^T) B_a^T.
//
// Three kernels.  The plan (once a step) sorts the tokens by adapter and cuts
// them into tiles of up to 64, so that an adapter's matrices are read once per
// tile and not once per token.  The shrink kernel computes h = x A^T of a tile
// over a part of in_features; the expand kernel adds the parts in order,
// splits s h into three bf16 (together its 24 bits: fp32 y keeps its accuracy),
// multiplies by B^T and adds y.  The products are m16n8k16: their operations
// take a small part of the bytes' time, and tiles of 1 to 64 tokens would leave
// most of a tcgen05 tile empty.  Bound by memory: the shrink by x
// (prompts) or A (decode), the expand by reading and writing y and by B; then
// by how evenly tiles of 1 to 64 tokens fill the SMs.  A call of 40 requests of
// up to 50 tokens, 24 adapters of rank 64, 4096 to 11008 features: 63 us,
// shrink 15 and expand 40 (bytes: 22; its warps wait for the loads of y and B); 6 prompts of up to 2048 tokens, rank 32,
// 11008 to 4096: 109 us, shrink 32 and expand 54 with 120 MB of x and y left in
// L2 by the call before (61); 64 decoding requests, rank 16, 4096 to 4096: 14 to 15 us, the calls and two launches.
#include "serving_common.cuh"

#include "tc_pipe.cuh"

namespace hxq {
namespace serving {

constexpr uint32_t kTile = HXQ_LORA_TILE;
constexpr int kLoraPlanThreads = 512;
constexpr int kShrinkRanks = 32;   // rows of A a CTA takes

// ---------------------------------------------------------------------------
// The plan: groups' sizes (one warp over the requests in order, so that tokens
// keep theirs), their tiles (block scans), then tiles and order, found by
// binary search.  Every CTA does the first two itself: one launch, 6 to 7 us for
// up to 64 requests; one warp takes 32 more of them a turn.
struct LoraPlanArgs {
    const int32_t *starts, *ids;
    int32_t *order;
    hxq_lora_tile_t *tiles;
    uint32_t *status;
    uint32_t B, n, T, n_tiles;
};

__global__ void __launch_bounds__(kLoraPlanThreads) lora_plan_kernel(const LoraPlanArgs a)
{
    // group n is that of tokens without an adapter
    extern __shared__ uint32_t sm[];
    uint32_t *count = sm, *first = count + a.n + 1, *tile = first + a.n + 1, *at = tile + a.n + 1, *from = at + a.B;
    __shared__ uint32_t wsum[2][kLoraPlanThreads / 32], carry[2];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (uint32_t i = tid; i <= a.n; i += kLoraPlanThreads) count[i] = 0;
    if (tid < 2) carry[tid] = 0;
    __syncthreads();
    let_next_start();
    // where a request's tokens go in its group: the group's tokens so far
    uint32_t bad = 0;
    if (warp == 0) {
        for (uint32_t b0 = 0; b0 < a.B; b0 += 32) {
            const uint32_t b = b0 + lane;
            uint32_t n = 0, group = a.n + 1;
            if (b < a.B) {
                const int32_t s = a.starts[b], e = a.starts[b + 1], id = a.ids[b];
                const uint32_t s0 = (uint32_t)min(max(s, 0), (int32_t)a.T), s1 = (uint32_t)min(max(e, (int32_t)s0), (int32_t)a.T);
                if (s < 0 || e < s || e > (int32_t)a.T) bad |= HXQ_SERVING_BAD_LENGTH;
                if (id >= (int32_t)a.n) bad |= HXQ_SERVING_BAD_ADAPTER;
                n = s1 - s0;
                group = id < 0 || id >= (int32_t)a.n ? a.n : (uint32_t)id;
                from[b] = s0;
            }
            const uint32_t same = __match_any_sync(~0u, group);
            uint32_t before = 0, all = 0;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const uint32_t v = __shfl_sync(~0u, n, k);
                if (same >> k & 1u) {
                    all += v;
                    if (k < (int)lane) before += v;
                }
            }
            const uint32_t so_far = group <= a.n ? count[group] : 0;
            __syncwarp();
            if (b < a.B) {
                at[b] = so_far + before;
                if ((same >> lane) == 1u) count[group] = so_far + all;   // the group's last lane
            }
            __syncwarp();
        }
        if (bad && blockIdx.x == 0) flag(a.status, bad);
    }
    __syncthreads();
    for (uint32_t g0 = 0; g0 <= a.n; g0 += kLoraPlanThreads) {
        const uint32_t i = g0 + tid, c = i <= a.n ? count[i] : 0, t = (c + kTile - 1) / kTile;
        uint32_t x = c, y = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t u = __shfl_up_sync(~0u, x, d), v = __shfl_up_sync(~0u, y, d);
            if (lane >= (uint32_t)d) { x += u; y += v; }
        }
        if (lane == 31) { wsum[0][warp] = x; wsum[1][warp] = y; }
        __syncthreads();
        uint32_t px = carry[0], py = carry[1];
        for (uint32_t w = 0; w < warp; ++w) { px += wsum[0][w]; py += wsum[1][w]; }
        x += px;
        y += py;
        if (i <= a.n) { first[i] = x - c; tile[i] = y - t; }
        __syncthreads();
        if (tid == kLoraPlanThreads - 1) { carry[0] = x; carry[1] = y; }
        __syncthreads();
    }
    const uint32_t used = carry[1];
    const uint32_t me = blockIdx.x * kLoraPlanThreads + tid, step = gridDim.x * kLoraPlanThreads;
    for (uint32_t i = me; i < a.n_tiles; i += step) {
        hxq_lora_tile_t t = {-1, 0, 0, 0};
        if (i < used) {
            uint32_t lo = 0, hi = a.n + 1;   // the last group whose first tile is at most i and that has tokens
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (tile[mid] <= i) lo = mid;
                else hi = mid;
            }
            const uint32_t off = (i - tile[lo]) * kTile;
            t.adapter = lo == a.n ? -1 : (int32_t)lo;
            t.first = (int32_t)(first[lo] + off);
            t.count = (int32_t)min(kTile, count[lo] - off);
        }
        a.tiles[i] = t;
    }
    for (uint32_t t = me; t < a.T; t += step) {
        uint32_t lo = 0, hi = a.B;   // the last request that begins at or before t
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (from[mid] <= t) lo = mid;
            else hi = mid;
        }
        if (a.B == 0 || t < from[lo]) continue;
        const int32_t e = a.starts[lo + 1];
        if ((int64_t)t >= (int64_t)e) continue;
        const int32_t id = a.ids[lo];
        const uint32_t group = id < 0 || id >= (int32_t)a.n ? a.n : (uint32_t)id;
        const uint32_t to = first[group] + at[lo] + (t - from[lo]);
        if (to < a.T) a.order[to] = (int32_t)t;   // always, unless starts descend
    }
}

// ---------------------------------------------------------------------------
struct LoraArgs {
    const uint16_t *x, *A, *Bm;
    const float *scales, *y;
    float *out, *h;              // h [parts][T][rank]: partial x A^T by sorted position
    const int32_t *order;
    const hxq_lora_tile_t *tiles;
    int64_t ldx, ldy, ldo;
    uint32_t T, n, R, I, O, parts, span;   // span: in_features of a part, a multiple of 128
    uint32_t pairs;                        // expand: pieces of 64 outputs a CTA takes
};

// A tile's positions come from device memory that the caller could have
// filled otherwise; keep them inside the arrays.
__device__ __forceinline__ bool load_tile(const LoraArgs &a, uint32_t i, int32_t &id, uint32_t &first, uint32_t &count)
{
    const int4 t = __ldg(reinterpret_cast<const int4 *>(a.tiles) + i);
    id = t.x;
    first = (uint32_t)t.y;
    count = (uint32_t)t.z;
    if (t.z <= 0 || t.y < 0 || first >= a.T || id >= (int32_t)a.n) return false;
    count = min(min(count, kTile), a.T - first);
    return true;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool wanted)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(wanted ? 16 : 0) : "memory");
}

constexpr int kShrinkRing = 24 * 1024;   // bytes of a warp's ring

// h[token, r] over [k0, k1) for 8 NT tokens: warps take 32 consecutive k in
// turn.  A lane holds 8 consecutive k of a row (16 bytes), the same ones of A
// and x, which are the operands of two m16n8k16 products; the pieces come
// through slots of shared memory that no other lane reads (cp.async, several
// steps ahead, no barrier): 24 KB a warp under way, two CTAs an SM.
template <int NT>
__device__ __forceinline__ void shrink_body(const LoraArgs &a, const uint16_t *A, uint32_t rows, const int64_t *xrow, uint32_t count,
                                            uint32_t k0, uint32_t k1, uint32_t ring, float (*red)[kShrinkRanks][kTile + 1])
{
    constexpr int kStep = (4 + NT) * 512, kStages = kShrinkRing / kStep < 8 ? kShrinkRing / kStep : 8;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const uint16_t *ap = A + (size_t)g * a.I, *xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = a.x + xrow[n * 8 + g];
    const uint32_t dst0 = ring + lane * 16;
    auto issue = [&](uint32_t k, uint32_t stage) {   // k: this lane's
        const uint32_t dst = dst0 + stage * kStep;
        const bool in = k < k1;
        const uint32_t kk = in ? k : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool w = in && i * 8 + g < rows;
            copy16(dst + i * 512, w ? ap + (size_t)i * 8 * a.I + kk : A, w);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) copy16(dst + (4 + n) * 512, xp[n] + kk, in && n * 8 + g < count);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.0f;
    const uint32_t first = k0 + warp * 32 + q * 8, steps = k0 + warp * 32 < k1 ? (k1 - k0 - warp * 32 + 127) / 128 : 0;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(first + i * 128, i);
    uint32_t stage = 0;
    for (uint32_t i = 0; i < steps; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        issue(first + (i + kStages - 1) * 128, stage == 0 ? kStages - 1 : stage - 1);
        const uint32_t src = dst0 + stage * kStep;
        uint4 av[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) av[r] = pipe::lds128(src + r * 512);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint4 xv = pipe::lds128(src + (4 + n) * 512);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                pipe::mma16816_bf16(acc[m][n], av[2 * m].x, av[2 * m + 1].x, av[2 * m].y, av[2 * m + 1].y, xv.x, xv.y);
                pipe::mma16816_bf16(acc[m][n], av[2 * m].z, av[2 * m + 1].z, av[2 * m].w, av[2 * m + 1].w, xv.z, xv.w);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // the four warps' sums: (0 + 2) + (1 + 3), the latter added by the caller
    auto each = [&](auto f) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) f(acc[m][n][e], m * 16 + g + (e >> 1) * 8, n * 8 + 2 * q + (e & 1));
    };
    if (warp >= 2) each([&](float v, int r, int t) { red[warp - 2][r][t] = v; });
    __syncthreads();
    if (warp < 2) each([&](float v, int r, int t) { red[warp][r][t] += v; });
    __syncthreads();
}

__global__ void __launch_bounds__(128, 2) shrink_kernel(const __grid_constant__ LoraArgs a)
{
    extern __shared__ __align__(128) uint8_t rings[];
    __shared__ float red[2][kShrinkRanks][kTile + 1];
    __shared__ int64_t xrow[kTile];
    wait_previous();
    let_next_start();   // not before: the next kernel reads y ahead of its own wait
    int32_t id;
    uint32_t first, count;
    if (!load_tile(a, blockIdx.x, id, first, count) || id < 0) return;
    const uint32_t tid = threadIdx.x;
    if (tid < kTile) {
        const int32_t t = tid < count ? a.order[first + tid] : 0;
        xrow[tid] = (int64_t)((uint32_t)t < a.T ? t : 0) * a.ldx;
    }
    __syncthreads();
    const uint32_t r0 = blockIdx.z * kShrinkRanks, rows = min((uint32_t)kShrinkRanks, a.R - r0);
    const uint16_t *A = a.A + ((size_t)id * a.R + r0) * a.I;
    const uint32_t k0 = blockIdx.y * a.span, k1 = min(k0 + a.span, a.I);
    const uint32_t ring = pipe::smem_u32(rings) + (tid >> 5) * kShrinkRing;
    if (count <= 8) shrink_body<1>(a, A, rows, xrow, count, k0, k1, ring, red);
    else if (count <= 16) shrink_body<2>(a, A, rows, xrow, count, k0, k1, ring, red);
    else if (count <= 32) shrink_body<4>(a, A, rows, xrow, count, k0, k1, ring, red);
    else shrink_body<8>(a, A, rows, xrow, count, k0, k1, ring, red);
    float *h = a.h + (size_t)blockIdx.y * a.T * a.R;
    for (uint32_t i = tid; i < count * rows; i += 128) {
        const uint32_t t = i / rows, r = i - t * rows;
        h[(size_t)(first + t) * a.R + r0 + r] = red[0][r][t] + red[1][r][t];
    }
}

__device__ __forceinline__ float4 load4(const float *p)
{
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float load1(const float *p)
{
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load2(const uint16_t *p)
{
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

__device__ __forceinline__ uint4 load_b(const uint16_t *p)
{
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// out = y + (s h) B^T: 16 tokens x 16 outputs at a time.  The two 8-output
// products of a piece take outputs {0,1,4,5,8,..} and {2,3,6,7,..}, so a lane
// ends with four consecutive outputs of a token (16-byte accesses of y).  A
// piece's B and y of the whole tile are loaded together, the first piece's
// before the shrink kernel's results are waited for.
template <int KS, bool WIDE> __global__ void __launch_bounds__(128, KS == 8 ? 2 : 4) expand_kernel(const __grid_constant__ LoraArgs a)
{
    // s h of the tile as operand fragments: [token group][k step][three parts][lane]
    extern __shared__ uint4 frag[];
    __shared__ int32_t rows[kTile];
    int32_t id;
    uint32_t first, count;
    if (!load_tile(a, blockIdx.x, id, first, count)) {
        wait_previous();
        return;
    }
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    if (tid < kTile) {
        const int32_t t = tid < count ? a.order[first + tid] : -1;
        rows[tid] = (uint32_t)t < a.T ? t : -1;
    }
    __syncthreads();
    // the CTA's warps side by side, so that it reads and writes 256 bytes of a
    // row of y at a time (64-byte pieces far apart: 2.5 times slower)
    const uint32_t o0 = (blockIdx.y * a.pairs * 4 + warp) * 16;
    if (id < 0) {
        // no adapter: out is y
        wait_previous();
        if (a.out == a.y && a.ldo == a.ldy) return;
        const uint32_t c0 = blockIdx.y * a.pairs * 64, n = min(a.pairs * 64, a.O > c0 ? a.O - c0 : 0);
        if (WIDE) {
            // 8 pieces of 16 bytes a thread under way
            const uint32_t per = n / 4, all = count * per;
            for (uint32_t i0 = tid; i0 < all; i0 += 128 * 8) {
                float4 v[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    const uint32_t i = i0 + u * 128, t = min(i, all - 1) / per;
                    v[u] = load4(a.y + (int64_t)max(rows[t], 0) * a.ldy + c0 + (min(i, all - 1) - t * per) * 4);
                }
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    const uint32_t i = i0 + u * 128, t = min(i, all - 1) / per;
                    if (i < all && rows[t] >= 0)
                        *reinterpret_cast<float4 *>(a.out + (int64_t)rows[t] * a.ldo + c0 + (i - t * per) * 4) = v[u];
                }
            }
        } else {
            for (uint32_t t = warp; t < count; t += 4) {
                if (rows[t] < 0) continue;
                const float *src = a.y + (int64_t)rows[t] * a.ldy + c0;
                float *dst = a.out + (int64_t)rows[t] * a.ldo + c0;
                for (uint32_t i = lane; i < n; i += 32) dst[i] = load1(src + i);
            }
        }
        return;
    }
    const uint32_t groups = (count + 15) / 16;
    const uint16_t *Bm = a.Bm + (size_t)id * a.O * a.R;
    uint2 b[2][2][KS];
    float4 y[2][4][2];   // two pieces: [token group][token g, g + 8]
    // loads that stay where they are written, all before the first use; a row
    // or column that does not exist reads one that does
    auto load = [&](uint32_t o, uint2 (&b)[2][KS], float4 (&y)[4][2]) {
        const uint32_t at = o + q * 4;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (m >= (int)groups) break;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int32_t tok = rows[m * 16 + g + 8 * r];
                const float *src = a.y + (int64_t)max(tok, 0) * a.ldy;
                if (WIDE) y[m][r] = load4(src + (at < a.O ? at : 0));
                else {
                    y[m][r].x = load1(src + min(at, a.O - 1));
                    y[m][r].y = load1(src + min(at + 1, a.O - 1));
                    y[m][r].z = load1(src + min(at + 2, a.O - 1));
                    y[m][r].w = load1(src + min(at + 3, a.O - 1));
                }
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t col = min(o + (g >> 1) * 4 + (g & 1) + 2 * w, a.O - 1);
            if (KS == 1) {
                b[w][0] = make_uint2(0, 0);
                if (q * 4 < a.R) b[w][0] = load2(Bm + (size_t)col * a.R + q * 4);
            } else {
                // 8 ranks a lane: two steps' operands
#pragma unroll
                for (int k = 0; k < KS; k += 2) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (k * 16 + q * 8 < a.R) v = load_b(Bm + (size_t)col * a.R + k * 16 + q * 8);
                    b[w][k] = make_uint2(v.x, v.y);
                    b[w][(k + 1) % KS] = make_uint2(v.z, v.w);
                }
            }
        }
    };
    const float scale = a.scales[id];
    if (o0 < a.O) load(o0, b[0], y[0]);
    wait_previous();
    for (uint32_t i = warp; i < groups * KS; i += 4) {
        const uint32_t m = i / KS, k = i % KS;
        uint32_t w3[3][4];
        float4 sums[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
        const uint32_t c = KS == 1 ? q * 4 : (k >> 1) * 32 + q * 8 + (k & 1) * 4, t0 = min(m * 16 + g, count - 1), t1 = min(m * 16 + g + 8, count - 1);
        const float *h0 = a.h + (size_t)(first + t0) * a.R + min(c, a.R - 4), *h1 = a.h + (size_t)(first + t1) * a.R + min(c, a.R - 4);
        for (uint32_t p0 = 0; p0 < a.parts; p0 += 4) {
            float4 u[4][2];
#pragma unroll
            for (uint32_t p = 0; p < 4; ++p) {
                const size_t off = (size_t)min(p0 + p, a.parts - 1) * a.T * a.R;
                u[p][0] = load4(h0 + off);
                u[p][1] = load4(h1 + off);
            }
#pragma unroll
            for (uint32_t p = 0; p < 4; ++p)
                if (p0 + p < a.parts)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        sums[r].x += u[p][r].x;
                        sums[r].y += u[p][r].y;
                        sums[r].z += u[p][r].z;
                        sums[r].w += u[p][r].w;
                    }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float4 v = sums[r];
            if (m * 16 + g + 8 * r >= count || c >= a.R) v = make_float4(0, 0, 0, 0);
            float f[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
            // (bf16 ends before fp32 does: what would round to an infinity, but is none, leaves the rest to the next parts)
            constexpr float kTopBf16 = 3.38953139e38f;
            auto top_of = [&](float x) { return fabsf(x) <= 3.402823466e38f ? fminf(fmaxf(x, -kTopBf16), kTopBf16) : x; };
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const __nv_bfloat162 top = part == 0 ? __floats2bfloat162_rn(top_of(f[2 * w]), top_of(f[2 * w + 1]))
                                                         : __floats2bfloat162_rn(f[2 * w], f[2 * w + 1]);
                    const float2 back = __bfloat1622float2(top);
                    // (nothing is left of an infinity)
                    f[2 * w] = fabsf(back.x) <= 3.402823466e38f ? f[2 * w] - back.x : 0.0f;
                    f[2 * w + 1] = fabsf(back.y) <= 3.402823466e38f ? f[2 * w + 1] - back.y : 0.0f;
                    w3[part][w * 2 + r] = *reinterpret_cast<const uint32_t *>(&top);
                }
        }
#pragma unroll
        for (int part = 0; part < 3; ++part)
            frag[(i * 3 + part) * 32 + lane] = make_uint4(w3[part][0], w3[part][1], w3[part][2], w3[part][3]);
    }
    __syncthreads();
    auto piece = [&](uint32_t o, const uint2 (&b)[2][KS], const float4 (&y)[4][2]) {
        const uint32_t at = o + q * 4;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (m >= (int)groups) break;
            float d[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int part = 2; part >= 0; --part) {
                    const uint4 h = frag[((m * KS + k) * 3 + part) * 32 + lane];
#pragma unroll
                    for (int w = 0; w < 2; ++w) pipe::mma16816_bf16(d[w], h.x, h.y, h.z, h.w, b[w][k].x, b[w][k].y);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int32_t tok = rows[m * 16 + g + 8 * r];
                if (tok < 0) continue;
                float *dst = a.out + (int64_t)tok * a.ldo + at;
                const float s[4] = {y[m][r].x + d[0][2 * r], y[m][r].y + d[0][2 * r + 1], y[m][r].z + d[1][2 * r],
                                    y[m][r].w + d[1][2 * r + 1]};
                if (WIDE) {
                    if (at < a.O) *reinterpret_cast<float4 *>(dst) = make_float4(s[0], s[1], s[2], s[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < a.O) dst[e] = s[e];
                }
            }
        }
    };
    // the next piece is on its way while this one is multiplied
    for (uint32_t j = 0; j < a.pairs; j += 2) {
        const uint32_t o = o0 + j * 64;
        if (o >= a.O) break;
        const bool more = j + 1 < a.pairs && o + 64 < a.O;
        if (more) load(o + 64, b[1], y[1]);
        piece(o, b[0], y[0]);
        if (!more) break;
        if (j + 2 < a.pairs && o + 128 < a.O) load(o + 128, b[0], y[0]);
        piece(o + 64, b[1], y[1]);
    }
}

template <int KS, bool WIDE> cudaError_t launch_expand(const LoraArgs &a, dim3 grid, cudaStream_t s)
{
    const size_t smem = (size_t)(kTile / 16) * KS * 3 * 32 * sizeof(uint4);
    static std::atomic<uint64_t> ready{0};
    if (smem > 40u * 1024u) {   // 48 KB with the kernel's static part need no permission
        const cudaError_t e = allow_smem(expand_kernel<KS, WIDE>, smem, ready);
        if (e != cudaSuccess) return e;
    }
    return launch_behind(expand_kernel<KS, WIDE>, grid, dim3(128), smem, s, a);
}

template <bool WIDE> cudaError_t launch_expand_rank(const LoraArgs &a, dim3 grid, cudaStream_t s)
{
    const uint32_t ks = (a.R + 15) / 16;
    return ks == 1 ? launch_expand<1, WIDE>(a, grid, s) : ks == 2 ? launch_expand<2, WIDE>(a, grid, s)
           : ks <= 4 ? launch_expand<4, WIDE>(a, grid, s) : launch_expand<8, WIDE>(a, grid, s);
}

// Parts that in_features is cut into, so that the shrink kernel has at least
// two CTAs for every SM; a part has at least 256 features.
uint32_t lora_parts(uint32_t tiles, uint32_t R, uint32_t I, uint32_t &span)
{
    const uint32_t blocks = tiles * ((R + kShrinkRanks - 1) / kShrinkRanks), want = 2u * (uint32_t)sm_count();
    uint32_t parts = blocks >= want ? 1u : (want + blocks - 1) / blocks;
    const uint32_t most = (I + 255) / 256;
    if (parts > most) parts = most;
    if (parts > 32) parts = 32;
    span = ((I + parts - 1) / parts + 127) / 128 * 128;
    return (I + span - 1) / span;
}

hxq_error_t check_lora(const hxq_lora_t *l)
{
    if (!l) return HXQ_ERR_NULL_PTR;
    if (l->n_adapters == 0 || l->n_adapters > HXQ_LORA_MAX_ADAPTERS) return HXQ_ERR_INVALID_ARG;
    if (l->rank == 0 || l->rank % 8 != 0 || l->rank > 128 || l->in_features == 0 || l->in_features % 8 != 0 ||
        l->out_features == 0 || l->in_features > 0x7fffff00u || l->out_features > 0x7fffff00u)
        return HXQ_ERR_INVALID_DIM;
    return HXQ_OK;
}

}  // namespace serving
}  // namespace hxq

using namespace hxq::serving;

extern "C" {

uint32_t hxq_lora_tiles(uint32_t B, uint32_t n_adapters, uint32_t n_tokens)
{
    const uint32_t groups = B < n_adapters ? B : n_adapters + 1;   // groups that can have tokens
    const uint64_t n = (uint64_t)n_tokens / HXQ_LORA_TILE + groups;
    return (uint32_t)(n < n_tokens ? n : n_tokens);
}

hxq_error_t hxq_cuda_lora_plan(const int32_t *d_starts, const int32_t *d_adapters, uint32_t B, uint32_t n_adapters,
                               uint32_t n_tokens, int32_t *d_order, hxq_lora_tile_t *d_tiles, uint32_t *d_status,
                               void *stream)
{
    if (B > HXQ_LORA_MAX_REQUESTS || n_adapters == 0 || n_adapters > HXQ_LORA_MAX_ADAPTERS || n_tokens > 0x7fffffffu)
        return HXQ_ERR_INVALID_ARG;
    if (n_tokens == 0 || B == 0) return HXQ_OK;
    if (!d_starts || !d_adapters || !d_order || !d_tiles) return HXQ_ERR_NULL_PTR;
    if (((uintptr_t)d_tiles & 15u) != 0) return HXQ_ERR_INVALID_ARG;
    LoraPlanArgs a = {d_starts, d_adapters, d_order, d_tiles, d_status, B, n_adapters, n_tokens,
                      hxq_lora_tiles(B, n_adapters, n_tokens)};
    const size_t smem = ((size_t)(n_adapters + 1) * 3 + (size_t)B * 2) * sizeof(uint32_t);
    const size_t most = ((size_t)(HXQ_LORA_MAX_ADAPTERS + 1) * 3 + (size_t)HXQ_LORA_MAX_REQUESTS * 2) * sizeof(uint32_t);
    static std::atomic<uint64_t> ready{0};
    if (smem > 40u * 1024u && allow_smem(lora_plan_kernel, most, ready) != cudaSuccess) {
        cudaGetLastError();
        return HXQ_ERR_CUDA;
    }
    const uint32_t want = (n_tokens + kLoraPlanThreads - 1) / kLoraPlanThreads, cap = (uint32_t)sm_count();
    lora_plan_kernel<<<want < cap ? want : cap, kLoraPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    return launched();
}

size_t hxq_cuda_lora_workspace(const hxq_lora_t *adapters, uint32_t n_requests, uint32_t n_tokens)
{
    if (check_lora(adapters) != HXQ_OK || n_tokens == 0) return 0;
    uint32_t span;
    const uint32_t tiles = hxq_lora_tiles(n_requests, adapters->n_adapters, n_tokens);
    return (size_t)lora_parts(tiles ? tiles : 1, adapters->rank, adapters->in_features, span) * n_tokens * adapters->rank * sizeof(float);
}

hxq_error_t hxq_cuda_lora(const hxq_lora_t *adapters, const uint16_t *d_x, int64_t ldx, const float *d_y, int64_t ldy,
                          float *d_out, int64_t ldo, uint32_t n_requests, uint32_t n_tokens, const int32_t *d_order,
                          const hxq_lora_tile_t *d_tiles, void *d_workspace, size_t workspace_bytes, void *stream)
{
    const hxq_error_t err = check_lora(adapters);
    if (err != HXQ_OK) return err;
    if (n_requests > HXQ_LORA_MAX_REQUESTS || n_tokens > 0x7fffffffu) return HXQ_ERR_INVALID_ARG;
    if (n_tokens == 0 || n_requests == 0) return HXQ_OK;
    if (!adapters->d_a || !adapters->d_b || !adapters->d_scales || !d_x || !d_y || !d_out || !d_order || !d_tiles || !d_workspace)
        return HXQ_ERR_NULL_PTR;
    if ((((uintptr_t)adapters->d_a | (uintptr_t)adapters->d_b | (uintptr_t)d_x | (uintptr_t)d_tiles | (uintptr_t)d_workspace) & 15u) != 0 ||
        (((uintptr_t)d_y | (uintptr_t)d_out) & 3u) != 0 || (ldx & 7) != 0)
        return HXQ_ERR_INVALID_ARG;
    const Runs out = {(uintptr_t)d_out, {n_tokens, 1}, {ldo, 0}, adapters->out_features, 4},
               y = {(uintptr_t)d_y, {n_tokens, 1}, {ldy, 0}, adapters->out_features, 4};
    if (!out.apart() || !out.may_overwrite(y)) return HXQ_ERR_INVALID_ARG;
    if (workspace_bytes < hxq_cuda_lora_workspace(adapters, n_requests, n_tokens)) return HXQ_ERR_INVALID_ARG;
    const uint32_t tiles = hxq_lora_tiles(n_requests, adapters->n_adapters, n_tokens);
    LoraArgs a;
    a.x = d_x;
    a.A = adapters->d_a;
    a.Bm = adapters->d_b;
    a.scales = adapters->d_scales;
    a.y = d_y;
    a.out = d_out;
    a.h = static_cast<float *>(d_workspace);
    a.order = d_order;
    a.tiles = d_tiles;
    a.ldx = ldx;
    a.ldy = ldy;
    a.ldo = ldo;
    a.T = n_tokens;
    a.n = adapters->n_adapters;
    a.R = adapters->rank;
    a.I = adapters->in_features;
    a.O = adapters->out_features;
    a.parts = lora_parts(tiles, a.R, a.I, a.span);
    // 16-byte accesses of y and out where every row allows them
    const bool wide = ((ldy | ldo | a.O) & 3) == 0 && (((uintptr_t)d_y | (uintptr_t)d_out) & 15u) == 0;
    // pieces of 64 outputs a CTA takes: 2 while that gives no more than four
    // CTAs an SM, up to 8 (tiles differ in length: some more CTAs than fit at
    // once even that out; one full wave of longer CTAs took a fifth more)
    const uint32_t pieces = (a.O + 63) / 64, full = 4u * (uint32_t)sm_count();
    a.pairs = 2;
    while (a.pairs < 8 && (uint64_t)tiles * ((pieces + a.pairs - 1) / a.pairs) > full) a.pairs *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid1(tiles, a.parts, (a.R + kShrinkRanks - 1) / kShrinkRanks);
    const dim3 grid2(tiles, (pieces + a.pairs - 1) / a.pairs);
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(shrink_kernel, 4 * kShrinkRing, ready);
    if (e == cudaSuccess) e = launch_behind(shrink_kernel, grid1, dim3(128), 4 * kShrinkRing, s, a);
    if (e == cudaSuccess) {
        e = wide ? launch_expand_rank<true>(a, grid2, s) : launch_expand_rank<false>(a, grid2, s);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return HXQ_ERR_CUDA;
    }
    return launched(2);
}

}  // extern "C"
