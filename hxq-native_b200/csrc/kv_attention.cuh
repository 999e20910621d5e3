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

cudaError_t launch_attn_mma(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, cudaStream_t s);
uint32_t attn_mma_ctas_per_sm(uint32_t D);

}  // namespace serving
}  // namespace hxq
