// kv_attention.cuh -- what the attention kernels over the 8-bit cache share:
// the request arithmetic and the code conversions.  Internal header.
#pragma once

#include "serving_common.cuh"

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
    uint32_t row_min, row_max;   // requests with row_min < rows <= row_max are this launch's
    float scale_log2;            // scale * log2(e)
    float *part;                 // partial results
    int4 *desc;                  // one per CTA
};

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
    const int64_t before = (int64_t)r.len - r.n;   // position of the request's first row
    lo = 0;
    hi = r.len;
    if (a.causal) {
        const int64_t last = before + (r1 - 1) / a.G + 1;
        hi = last < 0 ? 0u : last < (int64_t)r.len ? (uint32_t)last : r.len;
        if (a.window) {
            const int64_t first = before + r0 / a.G - (int64_t)a.window + 1;
            lo = first > 0 ? (uint32_t)first : 0u;
        }
    }
    if (lo > hi) lo = hi;
}

// The work of a launch: units (request, cache head, tile of ROWS rows) end to
// end, each as many granules of KEYS keys as its rows may see (one if none:
// the rows are written all the same), cut into one range for every CTA.
template <int ROWS, int KEYS> __device__ __forceinline__ uint32_t tile_grans(const AttnArgs &a, const Req &r, uint32_t t, uint32_t &first)
{
    uint32_t lo, hi;
    key_range(a, r, t * ROWS, min((t + 1) * ROWS, r.rows), lo, hi);
    first = lo / KEYS;
    const uint32_t last = (hi + KEYS - 1) / KEYS;
    return last > first ? last - first : 1u;
}

template <int ROWS, int KEYS> __device__ __forceinline__ uint64_t req_grans(const AttnArgs &a, const Req &r, uint32_t &most)
{
    uint64_t sum = 0;
    uint32_t first;
    for (uint32_t t = 0; t * ROWS < r.rows; ++t) {
        const uint32_t n = tile_grans<ROWS, KEYS>(a, r, t, first);
        sum += n;
        most = max(most, n);
    }
    return sum;
}

// Most parts of a unit that the joining kernel adds up.
constexpr uint32_t kMaxParts = 128;

template <int WARPS> struct RangeShared {
    uint64_t scan[WARPS];
    uint32_t most[WARPS];
    uint32_t b;
    uint64_t off;
};

// A position in the work: granule x of all, granule off of request b's.
struct Range {
    uint64_t x, x1, off, total, ctas;
    uint32_t b;
};

// This CTA's range, by a block scan over the requests; false: it has none.
// `record`: whether what is out of range is recorded (one launch of a call).
template <int WARPS, int ROWS, int KEYS>
__device__ __forceinline__ bool find_range(const AttnArgs &a, RangeShared<WARPS> &sh, bool record, Range &out)
{
    constexpr uint32_t N = WARPS * 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t per = (a.B + N - 1) / N, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    uint64_t mine = 0;
    uint32_t most = 1;
    for (uint32_t i = b0; i < b1; ++i) {
        mine += req_grans<ROWS, KEYS>(a, load_req(a, i), most) * a.H;
        if (record && blockIdx.x == 0) flag_req(a, i);
    }
    uint64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t u = __shfl_up_sync(~0u, incl, d);
        if (lane >= (uint32_t)d) incl += u;
    }
    most = __reduce_max_sync(~0u, most);
    if (lane == 31) {
        sh.scan[warp] = incl;
        sh.most[warp] = most;
    }
    if (tid == 0) { sh.b = a.B; sh.off = 0; }
    __syncthreads();
    uint64_t total = 0, before = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) {
        if (w < warp) before += sh.scan[w];
        total += sh.scan[w];
        most = max(most, sh.most[w]);
    }
    const uint64_t least = max(1u, (most + kMaxParts - 1) / kMaxParts);   // granules a CTA takes at least
    uint64_t n = (total + least - 1) / least;
    n = n < gridDim.x ? n : gridDim.x;
    if (blockIdx.x >= n) return false;
    out.x = total * blockIdx.x / n;
    out.x1 = total * (blockIdx.x + 1) / n;
    out.total = total;
    out.ctas = n;
    incl += before;
    if (incl - mine <= out.x && out.x < incl) {
        uint64_t at = incl - mine;
        for (uint32_t i = b0; i < b1; ++i) {
            const uint64_t w = req_grans<ROWS, KEYS>(a, load_req(a, i), most) * a.H;
            if (out.x < at + w) {
                sh.b = i;
                sh.off = out.x - at;
                break;
            }
            at += w;
        }
    }
    __syncthreads();
    out.b = sh.b;
    out.off = sh.off;
    return true;
}

// The part of a unit that a range has next.
struct Segment {
    Req r;
    uint32_t b, h, tile, first, rem, n, take, r0, r1, lo, hi;   // granules first + rem .. + take of the unit's n
};

template <int ROWS, int KEYS> __device__ __forceinline__ bool next_segment(const AttnArgs &a, Range &w, Segment &s)
{
    while (w.x < w.x1 && w.b < a.B) {
        s.r = load_req(a, w.b);
        uint32_t most = 0;
        const uint64_t sum = req_grans<ROWS, KEYS>(a, s.r, most);
        if (w.off >= sum * a.H) {
            w.off -= sum * a.H;
            ++w.b;
            continue;
        }
        s.b = w.b;
        s.h = (uint32_t)(w.off / sum);
        s.rem = (uint32_t)(w.off - s.h * sum);
        s.tile = 0;
        while (true) {
            s.n = tile_grans<ROWS, KEYS>(a, s.r, s.tile, s.first);
            if (s.rem < s.n) break;
            s.rem -= s.n;
            ++s.tile;
        }
        s.take = (uint32_t)min((uint64_t)(s.n - s.rem), w.x1 - w.x);
        s.r0 = s.tile * ROWS;
        s.r1 = min(s.r0 + ROWS, s.r.rows);
        key_range(a, s.r, s.r0, s.r1, s.lo, s.hi);
        w.x += s.take;
        w.off += s.take;
        return true;
    }
    return false;
}

// For the joining kernel, when a segment begins a unit and does not end it:
// how many ranges the unit lies in. (w is already behind the segment.)
__device__ __forceinline__ int4 cut_unit(const Range &w, const Segment &s)
{
    const uint64_t end = w.x - s.take + s.n;
    uint64_t c = blockIdx.x + 1;
    while (w.total * (c + 1) / w.ctas < end) ++c;
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
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// Weight of a value block: log2 of its scale (at least 2^-100), its inverse,
// and 0 or 1 for blocks that count as 0 or not.  NaN and infinity go through.
__device__ __forceinline__ void value_scale(float vs, float &lv, float &inv, bool &zero)
{
    zero = vs < 7.8886090522101181e-31f;   // 2^-100
    const float c = zero ? 7.8886090522101181e-31f : vs;
    lv = lg2(c);
    inv = __frcp_rn(c);
}

// Partial results of a CTA: two slots of ROWS x D sums, then the rows' maxima
// and sums; slot 0 a unit begun by the CTA in front, slot 1 one not finished.
template <int ROWS, int D> __host__ __device__ constexpr size_t part_floats() { return (size_t)ROWS * D + 2 * ROWS; }

// Joins the parts of the unit that CTA blockIdx.x began and did not finish:
// its own second slot, then the first slots of the CTAs behind it, in order.
// A warp takes a row.
template <int ROWS, int D, typename QT>
__device__ __forceinline__ void join_row(const AttnArgs &a, const int4 *desc, const float *parts, uint32_t cta, uint32_t rr)
{
    const int4 d = desc[cta];
    if (d.x == 0) return;
    const Req r = load_req(a, (uint32_t)d.y);
    const uint32_t row = (uint32_t)d.w * ROWS + rr, lane = threadIdx.x & 31;
    if (row >= r.rows) return;
    constexpr size_t kPart = part_floats<ROWS, D>();
    const float *first = parts + (2 * (size_t)cta + 1) * kPart, *rest = parts + 2 * ((size_t)cta + 1) * kPart;
    auto part = [&](int i) { return i == 0 ? first : rest + (size_t)(i - 1) * 2 * kPart; };
    float top = -INFINITY;
    for (int i = lane; i < d.x; i += 32) top = fmaxf(top, part(i)[ROWS * D + rr]);
#pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
    constexpr int N = D / 32;
    float v[N], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < d.x; ++i) {
        const float *p = part(i);
        const float m = p[ROWS * D + rr], w = top == -INFINITY ? 1.0f : ex2(m - top);
        sum += p[ROWS * D + ROWS + rr] * w;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += p[rr * D + j * 32 + lane] * w;
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t tok = r.q0 + row / a.G, head = (uint32_t)d.z * a.G + row % a.G;
    QT *dst = static_cast<QT *>(a.out) + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh;
#pragma unroll
    for (int j = 0; j < N; ++j) dst[j * 32 + lane] = Elem<QT>::from(v[j] * f);
    if (a.lse && lane == 0)
        a.lse[(size_t)tok * a.Hq + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

// Tensor-core kernel for many rows (kv_prefill.cu): launched behind the mma
// kernel of the same call; head_dim 64 or 128.
constexpr int kTcRows = 256;
cudaError_t launch_attn_tc(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, cudaStream_t s);

cudaError_t launch_attn_mma(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, bool join, cudaStream_t s);
uint32_t attn_mma_ctas_per_sm(uint32_t D);

}  // namespace serving
}  // namespace hxq
