// kv_attention.cuh -- what the attention kernels over the 8-bit cache share:
// the request arithmetic and the code conversions.  Internal header.
#pragma once

#include "serving_common.cuh"

#include "tc_pipe.cuh"

namespace hxq {
namespace serving {

struct AttnArgs {
    const void *q;
    void *out;
    float *lse;
    int64_t q_st, q_sh, o_st, o_sh;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *starts, *lens, *table;
    uint32_t *status;
    uint32_t B, T, Hq, H, G, P, n_blocks, width, window;
    uint32_t causal;
    uint32_t pmul;               // 2^32 / (P / 16), rounded up; 0 for P = 16
    uint32_t gmul;               // 2^32 / G, rounded up; 0 for G = 1
    uint32_t row_min, row_max;   // requests with row_min < rows <= row_max are this launch's
    float scale_log2;            // scale * log2(e)
    float *part;                 // partial results
    int4 *desc;                  // one per CTA
    uint32_t wait_cycles;        // most that a wait inside the kernel takes
};

// Wait for an mbarrier's phase, for at most a.wait_cycles cycles; false if
// they ran out, which is noted in gave_up (a word of shared memory), or if
// another wait of the CTA has noted it.
__device__ __forceinline__ bool bounded_wait(uint64_t *bar, uint32_t parity, uint32_t *gave_up, const AttnArgs &a)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 t0, t1;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE_%=;\n\tmov.u32 t0, %%clock;\n"
        "AGAIN_%=:\n\tmov.u32 t1, %%clock;\n\tsub.u32 t1, t1, t0;\n\tsetp.ge.u32 q, t1, %4;\n\t@q bra LATE_%=;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE_%=;\n\t"
        "ld.volatile.shared.u32 t1, [%3];\n\tsetp.ne.u32 q, t1, 0;\n\t@q bra DONE_%=;\n\tbra AGAIN_%=;\n"
        "LATE_%=:\n\tst.volatile.shared.u32 [%3], 1;\n"
        "DONE_%=:\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(pipe::smem_u32(bar)), "r"(parity), "r"(pipe::smem_u32(gave_up)), "r"(a.wait_cycles)
        : "memory");
    return ok != 0;
}

// For a thread that gave up on copies of its own: they end before the CTA does.
__device__ __forceinline__ void let_copies_end()
{
    const uint64_t t0 = clock64();
    while (clock64() - t0 < 20000000ull) {}
}

// One request: first q row, rows, keys; rows of a (request, cache head) are
// numbered token * G + group member.
struct Req {
    uint32_t q0, n, len, rows;
};

__device__ __forceinline__ Req load_req(const AttnArgs &a, uint32_t b)
{
    const int32_t s = __ldg(a.starts + b), e = __ldg(a.starts + b + 1), l = __ldg(a.lens + b);
    Req r;
    r.q0 = (uint32_t)min(max(s, 0), (int32_t)a.T);
    const uint32_t q1 = (uint32_t)min(max(e, (int32_t)r.q0), (int32_t)a.T);
    r.n = q1 - r.q0;
    const uint64_t most = (uint64_t)a.width * a.P;
    r.len = l < 0 ? 0u : (uint64_t)l > most ? (uint32_t)most : (uint32_t)l;
    r.rows = r.n * a.G;
    if (r.rows <= a.row_min || r.rows > a.row_max) r.rows = 0;
    return r;
}

// row / G: the product with the rounded-up inverse is right or one too large.
__device__ __forceinline__ uint32_t token_of(const AttnArgs &a, uint32_t row)
{
    if (a.gmul == 0) return row;
    const uint32_t q = __umulhi(row, a.gmul);
    return q - (q * a.G > row);
}

// Block of a request that a 16-aligned key is in, and its slot there
// (exact: key / 16 < 2^27, P / 16 <= 16).
__device__ __forceinline__ uint32_t block_of(const AttnArgs &a, uint32_t key, uint32_t &slot)
{
    const uint32_t k16 = key >> 4, b = a.pmul ? __umulhi(k16, a.pmul) : k16;
    slot = (k16 - b * (a.P >> 4)) << 4;
    return b;
}

// Called by one CTA of a launch: what was out of range is recorded.
__device__ __forceinline__ void flag_req(const AttnArgs &a, uint32_t b)
{
    const int32_t s = __ldg(a.starts + b), e = __ldg(a.starts + b + 1), l = __ldg(a.lens + b);
    if (s < 0 || e < s || e > (int32_t)a.T || l < 0) flag(a.status, HXQ_SERVING_BAD_LENGTH);
    if (l > 0 && (uint64_t)l > (uint64_t)a.width * a.P) flag(a.status, HXQ_SERVING_BAD_BLOCK);
}

// Keys [lo, hi) that rows r0 .. r1 - 1 of a request may see.
__device__ __forceinline__ void key_range(const AttnArgs &a, const Req &r, uint32_t r0, uint32_t r1, uint32_t &lo,
                                          uint32_t &hi)
{
    const int32_t before = (int32_t)r.len - (int32_t)r.n;   // position of the request's first row
    lo = 0;
    hi = r.len;
    if (a.causal) {
        const int32_t last = before + (int32_t)token_of(a, r1 - 1) + 1;
        hi = (uint32_t)min(max(last, 0), (int32_t)r.len);
        if (a.window) {
            const int64_t first = (int64_t)before + token_of(a, r0) - a.window + 1;
            lo = first > 0 ? (uint32_t)first : 0u;
        }
    }
    if (lo > hi) lo = hi;
}

// The work of a launch: units (request, cache head, tile of ROWS rows) end to
// end, each as many granules of KEYS keys as its rows may see (one if none:
// the rows are written all the same) behind FIXED ones that stand for the
// time a unit costs by itself, cut into one range for every CTA.
template <int ROWS, int KEYS> __device__ __forceinline__ uint32_t tile_grans(const AttnArgs &a, const Req &r, uint32_t t, uint32_t &first)
{
    uint32_t lo, hi;
    key_range(a, r, t * ROWS, min((t + 1) * ROWS, r.rows), lo, hi);
    first = lo / KEYS;
    const uint32_t last = (hi + KEYS - 1) / KEYS;
    return last > first ? last - first : 1u;
}

// Most parts of a unit that the joining kernel adds up.
constexpr uint32_t kMaxParts = 128;

template <int WARPS> struct RangeShared {
    uint64_t scan[WARPS];
    uint32_t most[WARPS];
    uint32_t b, tile;
    uint64_t off;
};

// A position in the work: granule x of all, up to x1 for this CTA; request b,
// tile, cache head h, granule rem of that unit's n.
struct Range {
    uint64_t x, x1, total, ctas;
    Req r;
    uint32_t b, tile, h, n, first, rem;
};

// This CTA's range; false: it has none. Requests' tiles are numbered through
// (a block scan, the sums in `pre`, B + 1 words of shared memory), then every
// thread counts the granules of some consecutive tiles (another scan), so a
// single long prompt is counted by all threads.  Heads of a tile follow each
// other.  `record`: whether what is out of range is recorded (one launch of a
// call).
template <int WARPS, int ROWS, int KEYS, int FIXED>
__device__ __forceinline__ bool find_range(const AttnArgs &a, RangeShared<WARPS> &sh, uint32_t *pre, bool record, Range &out)
{
    constexpr uint32_t N = WARPS * 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto scan = [&](uint64_t mine, uint64_t &total) {   // the sum in front of this thread
        uint64_t incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t u = __shfl_up_sync(~0u, incl, d);
            if (lane >= (uint32_t)d) incl += u;
        }
        if (lane == 31) sh.scan[warp] = incl;
        __syncthreads();
        uint64_t before = 0;
        total = 0;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) {
            if (w < warp) before += sh.scan[w];
            total += sh.scan[w];
        }
        return before + incl - mine;
    };
    uint64_t tiles;
    {
        const uint32_t per = (a.B + N - 1) / N, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
        uint64_t mine = 0;
        for (uint32_t i = b0; i < b1; ++i) {
            mine += (load_req(a, i).rows + ROWS - 1) / ROWS;
            if (record && blockIdx.x == 0) flag_req(a, i);
        }
        uint32_t at = (uint32_t)scan(mine, tiles);
        for (uint32_t i = b0; i < b1; ++i) {
            pre[i] = at;
            at += (load_req(a, i).rows + ROWS - 1) / ROWS;
        }
        if (tid == 0) { pre[a.B] = (uint32_t)tiles; sh.b = a.B; }
        __syncthreads();
    }
    // More than the rows there are make: starts that descend, so that requests overlap (recorded by flag_req). Their tiles
    // may be more than 32 bits count, and no program wants their work.
    if (tiles == 0 || tiles > (uint64_t)a.T * a.G / ROWS + a.B) return false;
    const uint32_t per = ((uint32_t)tiles + N - 1) / N, p0 = min(tid * per, (uint32_t)tiles), p1 = min(p0 + per, (uint32_t)tiles);
    uint32_t lo = 0, most = 1, first;
    uint64_t mine = 0;
    if (p0 < p1) {
        uint32_t hi = a.B;   // the last request with pre <= p0: it has tiles
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (pre[mid] <= p0) lo = mid;
            else hi = mid;
        }
        Req r = load_req(a, lo);
        for (uint32_t p = p0, b = lo; p < p1; ++p) {
            if (p >= pre[b + 1]) {
                while (p >= pre[b + 1]) ++b;
                r = load_req(a, b);
            }
            const uint32_t n = FIXED + tile_grans<ROWS, KEYS>(a, r, p - pre[b], first);
            mine += (uint64_t)n * a.H;
            most = max(most, n);
        }
    }
    most = __reduce_max_sync(~0u, most);
    if (lane == 31) sh.most[warp] = most;
    uint64_t at = scan(mine, out.total);
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) most = max(most, sh.most[w]);
    const uint64_t least = (most + kMaxParts - 1) / kMaxParts;   // granules a CTA takes at least
    uint64_t n = (out.total + least - 1) / least;
    n = n < gridDim.x ? n : gridDim.x;
    if (blockIdx.x >= n) return false;
    if (out.total <= 0xffffffffu / 4096u && gridDim.x < 4096u) {   // products of 32 bits
        out.x = (uint32_t)out.total * blockIdx.x / (uint32_t)n;
        out.x1 = (uint32_t)out.total * (blockIdx.x + 1) / (uint32_t)n;
    } else {
        out.x = out.total * blockIdx.x / n;
        out.x1 = out.total * (blockIdx.x + 1) / n;
    }
    out.ctas = n;
    if (at <= out.x && out.x < at + mine) {
        Req r = load_req(a, lo);
        for (uint32_t p = p0, b = lo; p < p1; ++p) {
            if (p >= pre[b + 1]) {
                while (p >= pre[b + 1]) ++b;
                r = load_req(a, b);
            }
            const uint64_t w = (uint64_t)(FIXED + tile_grans<ROWS, KEYS>(a, r, p - pre[b], first)) * a.H;
            if (out.x < at + w) {
                sh.b = b;
                sh.tile = p - pre[b];
                sh.off = out.x - at;
                break;
            }
            at += w;
        }
    }
    __syncthreads();
    out.b = sh.b;
    if (out.b >= a.B) return false;   // never: the ranges cover all granules
    out.tile = sh.tile;
    out.r = load_req(a, out.b);
    out.n = FIXED + tile_grans<ROWS, KEYS>(a, out.r, out.tile, out.first);
    out.h = sh.off <= 0xffffffffu ? (uint32_t)sh.off / out.n : (uint32_t)(sh.off / out.n);
    out.rem = (uint32_t)(sh.off - (uint64_t)out.h * out.n);
    return true;
}

// The part of a unit that a range has next.
struct Segment {
    Req r;
    uint32_t b, h, tile, key0, take, r0, r1, lo, hi, n;   // granules from key key0 on, of the unit's n
    bool begins;                                          // with the unit's first granule
    uint64_t end;                                         // of the unit, in the numbering of all granules
};

template <int ROWS, int KEYS, int FIXED> __device__ __forceinline__ bool next_segment(const AttnArgs &a, Range &w, Segment &s)
{
    while (w.x < w.x1 && w.b < a.B) {
        // granules of keys among those that are left, of the unit's n
        const uint32_t from = w.rem > FIXED ? w.rem - FIXED : 0u, step = (uint32_t)min((uint64_t)(w.n - w.rem), w.x1 - w.x);
        const uint32_t to = w.rem + step > FIXED ? w.rem + step - FIXED : 0u;
        s.r = w.r;
        s.b = w.b;
        s.h = w.h;
        s.tile = w.tile;
        s.n = w.n - FIXED;
        s.begins = from == 0;
        s.key0 = (w.first + from) * KEYS;
        s.take = to - from;
        w.x += step;
        w.rem += step;
        s.end = w.x + (w.n - w.rem);
        if (w.rem == w.n && w.x < w.x1) {
            w.rem = 0;
            if (++w.h == a.H) {
                w.h = 0;
                if (++w.tile * ROWS >= w.r.rows) {
                    w.tile = 0;
                    while (++w.b < a.B) {
                        w.r = load_req(a, w.b);
                        if (w.r.rows) break;
                    }
                }
                if (w.b < a.B) w.n = FIXED + tile_grans<ROWS, KEYS>(a, w.r, w.tile, w.first);
            }
        }
        if (s.take == 0) continue;   // the range ends before the unit's first keys: the next CTA begins it
        s.r0 = s.tile * ROWS;
        s.r1 = min(s.r0 + ROWS, s.r.rows);
        key_range(a, s.r, s.r0, s.r1, s.lo, s.hi);
        return true;
    }
    return false;
}

// For the joining kernel, when a segment begins a unit and does not end it:
// how many ranges, from this one on, the unit lies in.
__device__ __forceinline__ int4 cut_unit(const Range &w, const Segment &s)
{
    uint64_t c = blockIdx.x + 1;
    while (w.total * (c + 1) / w.ctas < s.end) ++c;
    return make_int4((int)(c - blockIdx.x + 1), (int)s.b, (int)s.h, (int)s.tile);
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x)
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 at a time.
__device__ __forceinline__ uint64_t pack2(float x, float y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v)
{
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(v));
    return d;
}

// Four codes of a word as f16 pairs (exact): int8 c becomes 1024 + (c + 128)
// by its bits, less 1152.
template <int FMT> __device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if (FMT == HXQ_KV_INT8) {
        w ^= 0x80808080u;
        lo = sub_f16x2(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u);
        hi = sub_f16x2(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u);
    } else {
        lo = e4m3x2_to_f16x2((uint16_t)w);
        hi = e4m3x2_to_f16x2((uint16_t)(w >> 16));
    }
}

// Weights are held times 2^kLift: f16 rounds below 2^-14 by 2^-25 whatever the
// size, which a lift of 7 puts at 2^-32 of a row's largest contribution.  With
// the largest at 2^0 a key that takes nearly all of the weight and has a small
// value left the others few bits (131,000 of them, 0.01 of the weight: a fifth
// of the output).  The largest weight before the maximum is raised is 2^15, f16
// holds 2^16.  Sums carry the factor, which the quotient drops.
constexpr float kLift = 7.0f;

// Weight of a value block: log2 of its scale (at least 2^-80), its inverse,
// and 0 or 1 for blocks that count as 0 or not.  NaN and infinity go through.
// The floor keeps 2^31 keys' 2^15 / vs within fp32.
__device__ __forceinline__ void value_scale(float vs, float &lv, float &inv, bool &zero)
{
    zero = vs < 8.271806125530277e-25f;   // 2^-80
    const float c = zero ? 8.271806125530277e-25f : vs;
    lv = lg2(c);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(c));   // within an ulp
}

// Partial results of a CTA: two slots of ROWS x D sums, then the rows' maxima
// and sums; slot 0 a unit begun by the CTA in front, slot 1 one not finished.
template <int ROWS, int D> __host__ __device__ constexpr size_t part_floats() { return (size_t)ROWS * D + 2 * ROWS; }

// Joins the parts of the unit that CTA `cta` began and did not finish: its own
// second slot, then the first slots of the CTAs behind it, in order.  A warp
// takes row rr of the unit's tile of ROWS (SLOT rows a slot); a lane looks
// after the weight of a part.
template <int ROWS, int SLOT, int D, int AHEAD, typename QT>
__device__ __forceinline__ void join_row(const AttnArgs &a, const int4 *desc, const float *parts, uint32_t cta, uint32_t rr)
{
    const int4 d = desc[cta];
    if (d.x == 0) return;
    constexpr size_t kPart = part_floats<SLOT, D>();
    constexpr int N = D / 32;
    const uint32_t lane = threadIdx.x & 31;
    const float *first = parts + (2 * (size_t)cta + 1) * kPart, *rest = parts + 2 * (size_t)cta * kPart;
    auto part = [&](int i) { return i == 0 ? first : rest + (size_t)i * 2 * kPart; };
    float v[N], u[AHEAD][N], sum = 0.0f;
    auto fetch = [&](int i0) {   // sums of AHEAD parts, N consecutive dimensions a lane
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) u[i][j] = 0.0f;
            if (i0 + i < d.x) {
                const float *p = part(i0 + i) + rr * D + lane * N;
                if constexpr (N == 2) {
                    const float2 f = *reinterpret_cast<const float2 *>(p);
                    u[i][0] = f.x;
                    u[i][1] = f.y;
                } else {
#pragma unroll
                    for (int j = 0; j < N; j += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(p + j);
                        u[i][j] = f.x;
                        u[i][j + 1] = f.y;
                        u[i][j + 2] = f.z;
                        u[i][j + 3] = f.w;
                    }
                }
            }
        }
    };
    // one latency for all of it: the first parts, their maxima and sums, the
    // request
    fetch(0);
    float t0 = -INFINITY, s0 = 0.0f;
    if ((int)lane < d.x) {
        const float *p = part(lane) + SLOT * D + rr;
        t0 = p[0];
        s0 = p[SLOT];
    }
    const Req r = load_req(a, (uint32_t)d.y);
    float top = t0;
    for (int i = lane + 32; i < d.x; i += 32) top = fmaxf(top, part(i)[SLOT * D + rr]);
#pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.0f;
    for (int i0 = 0; i0 < d.x; i0 += 32) {
        if (i0 > 0 && i0 + (int)lane < d.x) {
            const float *p = part(i0 + lane) + SLOT * D + rr;
            t0 = p[0];
            s0 = p[SLOT];
        }
        const float w = top == -INFINITY ? 1.0f : ex2(t0 - top);
#pragma unroll 1
        for (int k = 0; k < min(32, d.x - i0); k += AHEAD) {
            if (i0 + k > 0) fetch(i0 + k);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const float wi = __shfl_sync(~0u, w, k + i), si = __shfl_sync(~0u, s0, k + i);
                if (i0 + k + i < d.x) {
                    sum += si * wi;
#pragma unroll
                    for (int j = 0; j < N; ++j) v[j] += u[i][j] * wi;
                }
            }
        }
    }
    const uint32_t row = (uint32_t)d.w * ROWS + rr;
    if (row >= r.rows) return;
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t tk = token_of(a, row), tok = r.q0 + tk, head = (uint32_t)d.z * a.G + (row - tk * a.G);
    QT *dst = static_cast<QT *>(a.out) + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + lane * N;
    __align__(16) QT o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = Elem<QT>::from(v[j] * f);
    if (((uintptr_t)dst & (N * 2 - 1)) == 0) {
        if constexpr (N == 2) *reinterpret_cast<uint32_t *>(dst) = *reinterpret_cast<const uint32_t *>(o);
        else if constexpr (N == 4) *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(o);
        else *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(o);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) dst[j] = o[j];
    }
    if (a.lse && lane == 0)
        a.lse[(size_t)tok * a.Hq + head] = sum == 0.0f ? -INFINITY : (top - kLift + log2f(sum)) * 0.69314718055994531f;
}

// Tensor-core kernel for many rows (kv_prefill.cu): launched behind the mma
// kernel of the same call; head_dim 64 or 128.
constexpr int kTcRows = 256;
cudaError_t launch_attn_tc(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, cudaStream_t s);

// tc: the arguments of the kernel for many rows, where it runs too.
cudaError_t launch_attn_mma(const AttnArgs &a, const AttnArgs *tc, uint32_t D, uint32_t fmt, int elem, bool few, uint32_t grid, uint32_t tc_grid,
                            cudaStream_t s);

}  // namespace serving
}  // namespace hxq
