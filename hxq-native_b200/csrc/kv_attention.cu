// kv_attention.cu -- attention over the 8-bit cache for few query rows per
// key (decode, short chunks; any shape), and the C entry points.
//
// With S = q . code_k, a key's score is S * ks * scale and its value
// code_v * vs, ks and vs constant over a block.  In base 2, with
// lv = log2 vs, the weights exp2(s_j + lv_j - M) with M = max_j (s_j + lv_j)
// make both products run on codes alone:
//     out = sum_j w_j code_j / sum_j (w_j / vs_j),   0 <= w_j <= 1.
// Codes are exact in f16; w is rounded to f16 relative to the largest weighted
// contribution, so a block with large values and no weight costs the others
// nothing.  q is scaled per row by a power of two into f16's range (bf16
// values down to 2^-39 of the row's largest are exact).
//
// A CTA of four warps takes 16 rows (tokens x heads of a group) of one
// (request, cache head) against 64 keys at a time, 16 keys a warp: m16n8k16
// products, Q and the output accumulators in registers, every warp its own
// running maximum and sums, joined at the end of a segment.  A lane's share
// of a key row is 16 consecutive bytes: the order of the head's dimensions
// inside a product is free as long as Q has the same, so codes go from a
// lane's own 16-byte copies (cp.async into slots that no other lane reads: no
// barrier in the loop) through a byte permute into the fragments.
//
// The keys of all (request, head, 16 rows) are laid end to end in granules of
// 64 and cut into equal ranges, one per CTA; a range that ends inside a unit
// leaves a partial result (16 rows) in the workspace, and a second kernel
// joins the parts of each cut unit in order.  Every CTA derives the cut from
// the lengths itself, so it follows the lengths of a replayed graph.
#include "kv_attention.cuh"

#include "tc_pipe.cuh"

namespace hxq {
namespace serving {

constexpr int kRows = 16;        // rows of a tile
constexpr int kGran = 64;        // keys of a granule
constexpr int kFixed = 2;        // granules that a unit costs by itself
constexpr int kWarpsA = 4;
constexpr int kThreadsA = kWarpsA * 32;

template <int D> struct Geo {
    static constexpr int kVB = D >= 128 ? 16 : 8;      // bytes of a lane's copy of a value row
    static constexpr int kVC = D / (8 * kVB);          // copies of a value row per lane
    static constexpr int kKC = D / 64;                 // copies of a key row per lane
    static constexpr int kStepBytes = 32 * D;          // K and V of 16 keys
    static constexpr int kSlot = kStepBytes + 32 * 8;  // plus the two scales per lane
    static constexpr int kStages = D == 64 ? 6 : D == 128 ? 4 : 3;
    static constexpr int kQSmem = D == 256 ? 32 * D : 0;   // Q fragments in shared memory
    static constexpr int kRing = kWarpsA * kStages * kSlot;
    static constexpr int kPad = 4;
    static constexpr int kMerge = kWarpsA * kRows * (D + kPad) * 4;
    static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kQSmem;   // at least the scan's 4 (B + 1) bytes
    static_assert(kSmem >= 4 * (HXQ_ATTENTION_MAX_REQUESTS + 1), "room for the scan");
    static constexpr int kCtas = D == 256 ? 2 : 3;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void *src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename QT> __device__ __forceinline__ uint32_t to_f16x2(uint32_t w, float m)
{
    const QT *e = reinterpret_cast<const QT *>(&w);
    const __half2 h = __floats2half2_rn(Elem<QT>::to(e[0]) * m, Elem<QT>::to(e[1]) * m);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <int D, int FMT, typename QT>
__global__ void __launch_bounds__(kThreadsA, Geo<D>::kCtas) attn_mma_kernel(const __grid_constant__ AttnArgs a)
{
    using G = Geo<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RangeShared<kWarpsA> sh;
    __shared__ float sh_m[kWarpsA][kRows], sh_l[kWarpsA][kRows];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    let_next_start();

    if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    Range range;
    if (!find_range<kWarpsA, kRows, kGran, kFixed>(a, sh, reinterpret_cast<uint32_t *>(smem), true, range)) return;
    __syncthreads();   // the sums in front of the requests are read: the ring may be filled
    const uint32_t ring = pipe::smem_u32(smem) + warp * (G::kStages * G::kSlot);
    uint4 *qs = reinterpret_cast<uint4 *>(smem + (G::kSmem - G::kQSmem));
    float *merge = reinterpret_cast<float *>(smem);
    const uint32_t bh_bytes = a.P * D;

    Segment seg;
    while (next_segment<kRows, kGran, kFixed>(a, range, seg)) {
        const Req &r = seg.r;
        const uint32_t h = seg.h, take = seg.take, hi = seg.hi, r0 = seg.r0, r1 = seg.r1;
        const uint32_t key0 = seg.key0 + warp * 16;   // this warp's first 16 keys

        // ---- Q: rows g and g + 8, in the order in which codes arrive
        uint32_t qf[G::kQSmem ? 1 : D / 16][4];
        float fac[2];
        int32_t pos[2];
        {
            uint32_t raw[2][D / 16][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t row = r0 + g + 8 * i;
                const bool in = row < r1;
                const uint32_t tok = in ? token_of(a, row) : 0, head = h * a.G + (in ? row - tok * a.G : 0);
                pos[i] = in ? (a.causal ? (int32_t)((int64_t)r.len - r.n + tok) : (int32_t)r.len - 1) : -1;
                const QT *p = static_cast<const QT *>(a.q) + (int64_t)(r.q0 + tok) * a.q_st + (int64_t)head * a.q_sh;
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < G::kKC; ++c)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint4 v = in ? __ldg(reinterpret_cast<const uint4 *>(p + c * 64 + q * 16) + w)
                                           : make_uint4(0, 0, 0, 0);
                        raw[i][c * 4 + w * 2][0] = v.x;
                        raw[i][c * 4 + w * 2][1] = v.y;
                        raw[i][c * 4 + w * 2 + 1][0] = v.z;
                        raw[i][c * 4 + w * 2 + 1][1] = v.w;
                    }
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const QT *e = reinterpret_cast<const QT *>(&raw[i][s][w]);
                        top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[0]))));
                        top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[1]))));
                    }
                top = max(top, __shfl_xor_sync(~0u, top, 1));
                top = max(top, __shfl_xor_sync(~0u, top, 2));
                // 2^(14 - exponent of the largest): into [2^14, 2^15); 0 and non-finite rows as they are
                const int32_t e = (int32_t)(top >> 23) - 127;
                const int32_t sh = (top == 0 || e == 128) ? 0 : max(-100, min(100, 14 - e));
                const float m = __uint_as_float((uint32_t)(127 + sh) << 23);
                fac[i] = a.scale_log2 * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) raw[i][s][w] = to_f16x2<QT>(raw[i][s][w], m);
            }
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                if (G::kQSmem) {
                    if (warp == 0) qs[s * 32 + lane] = make_uint4(raw[0][s][0], raw[1][s][0], raw[0][s][1], raw[1][s][1]);
                } else {
                    qf[s % (G::kQSmem ? 1 : D / 16)][0] = raw[0][s][0];
                    qf[s % (G::kQSmem ? 1 : D / 16)][1] = raw[1][s][0];
                    qf[s % (G::kQSmem ? 1 : D / 16)][2] = raw[0][s][1];
                    qf[s % (G::kQSmem ? 1 : D / 16)][3] = raw[1][s][1];
                }
            }
            if (G::kQSmem) __syncthreads();
        }
        const int32_t pos_first = a.causal ? (int32_t)((int64_t)r.len - r.n + token_of(a, r0)) : (int32_t)r.len - 1;
        const int32_t pos_last = a.causal ? (int32_t)((int64_t)r.len - r.n + token_of(a, r1 - 1)) : (int32_t)r.len - 1;
        // a row sees keys above its floor: its position less the window, -1 without one
        auto key_floor = [&](int32_t at) { return a.window ? (int32_t)max((int64_t)at - (int64_t)a.window, (int64_t)-1) : -1; };
        const int32_t floor_last = key_floor(pos_last), floors[2] = {key_floor(pos[0]), key_floor(pos[1])};

        // ---- key loop
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        uint32_t valid = 0;   // bit s: the step in stage s has a block inside the cache
        const int32_t *row = a.table + (size_t)seg.b * a.width;
        auto entry = [&](uint32_t j) -> int32_t {
            const uint32_t key = key0 + j * kGran;
            uint32_t slot;
            return j < take && key < hi ? __ldg(row + block_of(a, key, slot)) : -1;
        };
        auto issue = [&](uint32_t j, uint32_t stage, int32_t blk) {
            const uint32_t key = key0 + j * kGran;
            const bool wanted = j < take && key < hi;
            const bool ok = wanted && (uint32_t)blk < a.n_blocks;
            if (wanted && !ok && lane == 0) flag(a.status, HXQ_SERVING_BAD_BLOCK);
            valid = ok ? valid | 1u << stage : valid & ~(1u << stage);
            if (ok) {
                const size_t bh = (size_t)(uint32_t)blk * a.H + h;
                uint32_t slot;
                block_of(a, key, slot);
                const size_t base = bh * bh_bytes + (size_t)slot * D;
                const uint32_t dst = ring + stage * G::kSlot + lane * 16;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int c = 0; c < G::kKC; ++c)
                        cp16(dst + (nt * G::kKC + c) * 512, a.k + base + (nt * 8 + g) * D + c * 64 + q * 16);
                const uint32_t vdst = ring + stage * G::kSlot + 16 * D + lane * G::kVB;
#pragma unroll
                for (int ts = 0; ts < 4; ++ts)
#pragma unroll
                    for (int c = 0; c < G::kVC; ++c) {
                        const void *src = a.v + base + (2 * q + (ts & 1) + (ts >> 1) * 8) * D + c * 128 + g * G::kVB;
                        if (G::kVB == 16) cp16(vdst + (ts * G::kVC + c) * 512, src);
                        else cp8(vdst + ts * 256, src);
                    }
                const uint32_t sdst = ring + stage * G::kSlot + 32 * D + lane * 8;
                cp4(sdst, a.ks + bh);
                cp4(sdst + 4, a.vs + bh);
            }
            cp_commit();
        };
        {
            int32_t blk[G::kStages - 1];
#pragma unroll
            for (int s = 0; s < G::kStages - 1; ++s) blk[s] = entry(s);
#pragma unroll
            for (int s = 0; s < G::kStages - 1; ++s) issue(s, s, blk[s]);
        }
        int32_t next = entry(G::kStages - 1);
        uint32_t stage = 0;
        for (uint32_t j = 0; j < take; ++j) {
            cp_wait<G::kStages - 2>();
            const bool live = valid >> stage & 1u;
            {
                const uint32_t into = stage == 0 ? G::kStages - 1 : stage - 1;
                issue(j + G::kStages - 1, into, next);
                next = entry(j + G::kStages);
            }
            if (live) {
                const uint32_t src = ring + stage * G::kSlot;
                const uint2 sc = pipe::lds64(src + 32 * D + lane * 8);
                float s[2][4];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
                    for (int c = 0; c < G::kKC; ++c) {
                        const uint4 kw = pipe::lds128(src + (nt * G::kKC + c) * 512 + lane * 16);
                        const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t b0, b1;
                            codes_to_f16<FMT>(w[i], b0, b1);
                            if (G::kQSmem) {
                                const uint4 f = qs[(c * 4 + i) * 32 + lane];
                                pipe::mma16816_f16(s[nt], f.x, f.y, f.z, f.w, b0, b1);
                            } else {
                                uint32_t *f = qf[(c * 4 + i) % (G::kQSmem ? 1 : D / 16)];
                                pipe::mma16816_f16(s[nt], f[0], f[1], f[2], f[3], b0, b1);
                            }
                        }
                    }
                }
                const uint32_t key = key0 + j * kGran;
                float lv, inv;
                bool zero;
                value_scale(__uint_as_float(sc.y), lv, inv, zero);
                const float ks = __uint_as_float(sc.x);
                const bool all = (int32_t)(key + 15) <= pos_first && (int32_t)key > floor_last && r1 - r0 == kRows;
                float top[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = fac[i] * ks;
                    top[i] = -INFINITY;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float t = fmaf(s[nt][2 * i + e], f, lv);
                            if (!all) {
                                const int32_t kp = (int32_t)(key + nt * 8 + 2 * q + e);
                                if (kp > pos[i] || kp <= floors[i]) t = -INFINITY;
                            }
                            s[nt][2 * i + e] = t;
                            top[i] = fmaxf(top[i], t);
                        }
                    top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 2));
                }
                if (__any_sync(~0u, top[0] > m[0] || top[1] > m[1])) {
                    float al[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float to = fmaxf(m[i], top[i]);
                        al[i] = to == -INFINITY ? 1.0f : ex2(m[i] - to);
                        m[i] = to;
                        l[i] *= al[i];
                    }
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        o[i][0] *= al[0];
                        o[i][1] *= al[0];
                        o[i][2] *= al[1];
                        o[i][3] *= al[1];
                    }
                }
                uint32_t p[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ms = m[i] == -INFINITY ? 0.0f : m[i];
                    float sum = 0.0f;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const float w0 = ex2(s[nt][2 * i] - ms), w1 = ex2(s[nt][2 * i + 1] - ms);
                        sum += w0 + w1;
                        const __half2 hh = __floats2half2_rn(w0, w1);
                        p[nt * 2 + i] = zero ? 0u : *reinterpret_cast<const uint32_t *>(&hh);
                    }
                    // a row that sees none of these keys takes nothing from the block, whatever its scale
                    l[i] += (sum == 0.0f) ? 0.0f : sum * inv;
                }
                const bool tail = key + 16 > hi;
#pragma unroll
                for (int c = 0; c < G::kVC; ++c) {
                    uint32_t vw[4][4];
#pragma unroll
                    for (int ts = 0; ts < 4; ++ts) {
                        if (G::kVB == 16) {
                            const uint4 v = pipe::lds128(src + 16 * D + (ts * G::kVC + c) * 512 + lane * 16);
                            vw[ts][0] = v.x;
                            vw[ts][1] = v.y;
                            vw[ts][2] = v.z;
                            vw[ts][3] = v.w;
                        } else {
                            const uint2 v = pipe::lds64(src + 16 * D + ts * 256 + lane * 8);
                            vw[ts][0] = v.x;
                            vw[ts][1] = v.y;
                            vw[ts][2] = vw[ts][3] = 0;
                        }
                        // slots behind the last key may hold anything
                        if (tail && key + 2 * q + (ts & 1) + (ts >> 1) * 8 >= hi)
                            vw[ts][0] = vw[ts][1] = vw[ts][2] = vw[ts][3] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < G::kVB / 4; ++i)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            // bytes 2 half, 2 half + 1 of two keys: (a, b, a, b)
                            const uint32_t sel = half ? 0x7362 : 0x5140;
                            uint32_t b0, b1, b2, b3;
                            codes_to_f16<FMT>(__byte_perm(vw[0][i], vw[1][i], sel), b0, b2);
                            codes_to_f16<FMT>(__byte_perm(vw[2][i], vw[3][i], sel), b1, b3);
                            const int t = c * G::kVB + i * 4 + half * 2;
                            pipe::mma16816_f16(o[t], p[0], p[1], p[2], p[3], b0, b1);
                            pipe::mma16816_f16(o[t + 1], p[0], p[1], p[2], p[3], b2, b3);
                        }
                }
            }
            stage = stage == G::kStages - 1 ? 0 : stage + 1;
        }
        cp_wait<0>();

        // ---- join the four warps
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(~0u, l[i], 1);
            l[i] += __shfl_xor_sync(~0u, l[i], 2);
            if (q == 0) {
                sh_m[warp][g + 8 * i] = m[i];
                sh_l[warp][g + 8 * i] = l[i];
            }
        }
        __syncthreads();
        float wt[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarpsA; ++w) top = fmaxf(top, sh_m[w][g + 8 * i]);
            wt[i] = top == -INFINITY ? 1.0f : ex2(m[i] - top);
        }
        float *mine = merge + warp * kRows * (D + G::kPad);
#pragma unroll
        for (int t = 0; t < D / 8; ++t) {
            const int d = (t / G::kVB) * 128 + (t % G::kVB);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mine[(g + (e >> 1) * 8) * (D + G::kPad) + d + (2 * q + (e & 1)) * G::kVB] = o[t][e] * wt[e >> 1];
        }
        __syncthreads();
        const bool whole = seg.begins && take == seg.n;
        float *part = a.part + (size_t)(2 * blockIdx.x + (seg.begins ? 1 : 0)) * part_floats<kRows, D>();
        for (uint32_t i = tid; i < kRows * (D / 4); i += kThreadsA) {
            const uint32_t rr = i / (D / 4), d = (i % (D / 4)) * 4;
            if (r0 + rr >= r1) break;
            float4 v = make_float4(0, 0, 0, 0);
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarpsA; ++w) {
                const float4 u = *reinterpret_cast<const float4 *>(merge + (w * kRows + rr) * (D + G::kPad) + d);
                v.x += u.x;
                v.y += u.y;
                v.z += u.z;
                v.w += u.w;
                top = fmaxf(top, sh_m[w][rr]);
            }
#pragma unroll
            for (int w = 0; w < kWarpsA; ++w) sum += top == -INFINITY ? sh_l[w][rr] : sh_l[w][rr] * ex2(sh_m[w][rr] - top);
            if (whole) {
                const uint32_t tk = token_of(a, r0 + rr), tok = r.q0 + tk, head = h * a.G + (r0 + rr - tk * a.G);
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                QT *dst = static_cast<QT *>(a.out) + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + d;
                dst[0] = Elem<QT>::from(v.x * f);
                dst[1] = Elem<QT>::from(v.y * f);
                dst[2] = Elem<QT>::from(v.z * f);
                dst[3] = Elem<QT>::from(v.w * f);
                if (a.lse && d == 0)
                    a.lse[(size_t)tok * a.Hq + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
            } else {
                *reinterpret_cast<float4 *>(part + rr * D + d) = v;
                if (d == 0) {
                    part[kRows * D + rr] = top;
                    part[kRows * D + kRows + rr] = sum;
                }
            }
        }
        if (seg.begins && take < seg.n && tid == 0) a.desc[blockIdx.x] = cut_unit(range, seg);
        __syncthreads();   // the ring is free again
    }
}

template <int D, typename QT> __global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs a)
{
    wait_previous();
    join_row<kRows, D, QT>(a, a.desc, a.part, blockIdx.x, blockIdx.y * 4 + (threadIdx.x >> 5));
}

template <int D, int FMT, typename QT> cudaError_t launch_one(const AttnArgs &a, uint32_t grid, bool join, cudaStream_t s)
{
    auto kernel = attn_mma_kernel<D, FMT, QT>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(kernel, Geo<D>::kSmem, ready);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kThreadsA, Geo<D>::kSmem, s>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess || !join) return e;
    return launch_behind(attn_join_kernel<D, QT>, dim3(grid, kRows / 4), dim3(128), 0, s, a);
}

template <int D> cudaError_t launch_dim(const AttnArgs &a, uint32_t fmt, int elem, uint32_t grid, bool join, cudaStream_t s)
{
    if (elem == HXQ_ELEM_BF16)
        return fmt == HXQ_KV_INT8 ? launch_one<D, HXQ_KV_INT8, __nv_bfloat16>(a, grid, join, s)
                                  : launch_one<D, HXQ_KV_E4M3, __nv_bfloat16>(a, grid, join, s);
    return fmt == HXQ_KV_INT8 ? launch_one<D, HXQ_KV_INT8, __half>(a, grid, join, s)
                              : launch_one<D, HXQ_KV_E4M3, __half>(a, grid, join, s);
}

cudaError_t launch_attn_mma(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, bool join, cudaStream_t s)
{
    return D == 64 ? launch_dim<64>(a, fmt, elem, grid, join, s)
                   : D == 128 ? launch_dim<128>(a, fmt, elem, grid, join, s) : launch_dim<256>(a, fmt, elem, grid, join, s);
}

uint32_t attn_mma_ctas_per_sm(uint32_t D)
{
    return D == 256 ? Geo<256>::kCtas : Geo<128>::kCtas;
}

hxq_error_t check_attention(const hxq_kv_cache_t *c, const hxq_kv_attention_t *p)
{
    const hxq_error_t err = check_cache(c);
    if (err != HXQ_OK) return err;
    if (!p) return HXQ_ERR_NULL_PTR;
    if (p->elem != HXQ_ELEM_BF16 && p->elem != HXQ_ELEM_F16) return HXQ_ERR_INVALID_ARG;
    if (p->n_heads == 0 || p->n_heads % c->n_heads != 0 || p->n_heads > 65535u) return HXQ_ERR_INVALID_DIM;
    if (p->n_requests > HXQ_ATTENTION_MAX_REQUESTS || (uint64_t)p->n_rows * (p->n_heads / c->n_heads) >= (1ull << 30))
        return HXQ_ERR_INVALID_ARG;
    if ((uint64_t)p->table_width * c->block_tokens >= (1ull << 31)) return HXQ_ERR_INVALID_ARG;
    if (p->window && !p->causal) return HXQ_ERR_INVALID_ARG;
    if (!(p->scale >= 0.0f) || p->scale > 3.402823466e38f) return HXQ_ERR_INVALID_ARG;
    return HXQ_OK;
}

// Workspace: a word group for every CTA, then the partial results, of this
// kernel and of the one for many rows.
struct AttnLayout {
    uint32_t ctas, tc_ctas;
    size_t part, tc_desc, tc_part, bytes;
};

// Requests with more rows than this go to the tcgen05 kernel.
constexpr uint32_t kFewRows = 64;

AttnLayout attn_layout(uint32_t D, uint64_t most_rows)
{
    AttnLayout l;
    const uint32_t sms = (uint32_t)sm_count();
    l.ctas = sms * attn_mma_ctas_per_sm(D);
    l.tc_ctas = D != 256 && most_rows > kFewRows ? sms : 0;
    l.part = l.ctas * sizeof(int4);
    l.tc_desc = l.part + (size_t)l.ctas * 2 * (kRows * D + 2 * kRows) * sizeof(float);
    l.tc_part = l.tc_desc + l.tc_ctas * sizeof(int4);
    l.bytes = l.tc_part + (size_t)l.tc_ctas * 2 * (kTcRows * D + 2 * kTcRows) * sizeof(float);
    return l;
}

}  // namespace serving
}  // namespace hxq

using namespace hxq::serving;

extern "C" {

size_t hxq_cuda_kv_attention_workspace(const hxq_kv_cache_t *cache, const hxq_kv_attention_t *args)
{
    if (check_attention(cache, args) != HXQ_OK) return 0;
    return attn_layout(cache->head_dim, (uint64_t)args->max_new * (args->n_heads / cache->n_heads)).bytes;
}

hxq_error_t hxq_cuda_kv_attention(const hxq_kv_cache_t *cache, const hxq_kv_attention_t *args, void *d_workspace,
                                  size_t workspace_bytes, uint32_t *d_status, void *stream)
{
    const hxq_error_t err = check_attention(cache, args);
    if (err != HXQ_OK) return err;
    if (args->n_requests == 0 || args->n_rows == 0) return HXQ_OK;
    if (!args->d_q || !args->d_out || !args->d_starts || !args->d_lens || !d_workspace || (!args->d_table && args->table_width))
        return HXQ_ERR_NULL_PTR;
    if ((((uintptr_t)args->d_q | (uintptr_t)d_workspace) & 15u) != 0 || ((args->q_stride_t | args->q_stride_h) & 7) != 0 ||
        ((uintptr_t)args->d_out & 1u) != 0)
        return HXQ_ERR_INVALID_ARG;
    const AttnLayout lay = attn_layout(cache->head_dim, (uint64_t)args->max_new * (args->n_heads / cache->n_heads));
    if (workspace_bytes < lay.bytes) return HXQ_ERR_INVALID_ARG;
    AttnArgs a;
    a.q = args->d_q;
    a.out = args->d_out;
    a.lse = args->d_lse;
    a.q_st = args->q_stride_t;
    a.q_sh = args->q_stride_h;
    a.o_st = args->out_stride_t;
    a.o_sh = args->out_stride_h;
    a.k = static_cast<const uint8_t *>(cache->k);
    a.v = static_cast<const uint8_t *>(cache->v);
    a.ks = cache->k_scales;
    a.vs = cache->v_scales;
    a.starts = args->d_starts;
    a.lens = args->d_lens;
    a.table = args->d_table;
    a.status = d_status;
    a.B = args->n_requests;
    a.T = args->n_rows;
    a.Hq = args->n_heads;
    a.H = cache->n_heads;
    a.G = args->n_heads / cache->n_heads;
    a.P = cache->block_tokens;
    a.pmul = a.P == 16 ? 0u : (uint32_t)(((1ull << 32) + a.P / 16 - 1) / (a.P / 16));
    a.gmul = a.G == 1 ? 0u : (uint32_t)(((1ull << 32) + a.G - 1) / a.G);
    a.n_blocks = cache->n_blocks;
    a.width = args->table_width;
    a.window = args->window;
    a.causal = args->causal != 0;
    a.row_min = 0;
    a.row_max = 0xffffffffu;
    a.scale_log2 = args->scale * 1.4426950408889634f;
    uint8_t *ws = static_cast<uint8_t *>(d_workspace);
    a.desc = reinterpret_cast<int4 *>(ws);
    a.part = reinterpret_cast<float *>(ws + lay.part);
    // Few rows of a request: this file's kernel. More: the tcgen05 kernel (64
    // is where a tile of 16 rows reads the keys four times over; that kernel
    // takes 128 rows at a time). Without rows of the other kind a launch ends
    // after its scan of the lengths.
    if (lay.tc_ctas) a.row_max = kFewRows;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_attn_mma(a, cache->head_dim, cache->format, args->elem, lay.ctas, true, s);
    if (e == cudaSuccess && lay.tc_ctas) {
        a.row_min = kFewRows;
        a.row_max = 0xffffffffu;
        a.desc = reinterpret_cast<int4 *>(ws + lay.tc_desc);
        a.part = reinterpret_cast<float *>(ws + lay.tc_part);
        e = launch_attn_tc(a, cache->head_dim, cache->format, args->elem, lay.tc_ctas, s);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return HXQ_ERR_CUDA;
    }
    return launched(lay.tc_ctas ? 4 : 2);
}

}  // extern "C"
