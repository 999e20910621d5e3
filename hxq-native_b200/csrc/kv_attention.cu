// kv_attention.cu -- attention over the 8-bit cache for few query rows per
// key (decode, short chunks; any shape), and the C entry points.
//
// With S = q . code_k, a key's score is S * ks * scale and its value
// code_v * vs, ks and vs constant over a block.  In base 2, with
// lv = log2 vs, the weights exp2(s_j + lv_j - M) with M = max_j (s_j + lv_j)
// make both products run on codes alone:
//     out = sum_j w_j code_j / sum_j (w_j / vs_j),   0 <= w_j <= 1.
// Codes are exact in f16; w (times 2^7) is rounded to f16 relative to the
// largest weighted contribution, so a block with large values and no weight
// costs the others nothing.  q is scaled per row by a power of two into f16's range (bf16
// values down to 2^-31 of the row's largest are exact).
//
// A CTA of four warps takes 8 or 16 rows (tokens x heads of a group) of one
// (request, cache head) against 64 keys at a time, 16 keys a warp, every warp
// with its own running maximum and sums, joined at the end of a segment.  The
// products are m16n8k16 with keys, then dimensions, on the side of 16 and rows
// on that of 8 (S^T = K Q^T, O^T = V^T P^T): one request's group of heads
// fills the small side, so a decode step of up to 8 heads a group wastes
// nothing of it.  TMA brings 16 keys' codes at a time (two boxes of 16 rows,
// swizzled so that the fragments' loads meet no bank twice) into a ring of each
// warp's own, two steps ahead; the order of the head's dimensions inside a
// product is free as long as Q has the same, so a lane reads 16 consecutive
// bytes of a key and brings them through a byte permute
// into the fragments; the weights turn round with movmatrix.  The maximum is
// raised only where a weight would grow by more than 2^8: a vote a step
// instead of a reduction.
//
// The keys of all (request, head, tile of rows) are laid end to end in granules of
// 64 and cut into equal ranges, one per CTA; a range that ends inside a unit
// leaves a partial result (16 rows) in the workspace, and a second kernel
// joins the parts of each cut unit in order.  Every CTA derives the cut from
// the lengths itself, so it follows the lengths of a replayed graph.
//
// Bound by instructions, then memory: 64 requests of up to 8192 keys, 8 heads of
// 128, groups of 4: 113 to 117 us a call, 71 to 73% of the copy bandwidth; 2 of
// 131,001 keys: 109 us, 75% (cp.async in place of TMA: 130 and 126; 8 rows on
// the side of 16: 166 and 158).  Instructions are issued in 58% of a scheduler's
// cycles and shared memory is at 56% of its wavefronts; a warp that waits does
// so for a fixed latency or shared memory, a seventh as often for device memory.  One request of
// 1024 keys takes 14.4 us a call, latency: launch, cut, copies, join.
#include "kv_attention.cuh"

#include "tc_pipe.cuh"

#include <type_traits>

namespace hxq {
namespace serving {

constexpr int kMostRows = 16;    // rows of a partial result's slot; a tile has 8 NT of them
constexpr int kGran = 64;        // keys of a granule
constexpr int kFixed = 2;        // granules that a unit costs by itself
constexpr int kWarpsA = 4;
constexpr int kThreadsA = kWarpsA * 32;
constexpr float kRaiseA = 8.0f;  // log2 of the largest weight (less the lift) before the maximum is raised

template <int D> struct Geo {
    static constexpr int kVB = D >= 128 ? 16 : 8;      // bytes of a lane's load of a value row
    static constexpr int kVC = D / (8 * kVB);          // loads of a value row per lane
    static constexpr int kKC = D / 64;                 // loads of a key row per lane
    static constexpr int kLine = D >= 128 ? 128 : 64;  // bytes of a box's rows (swizzled over that span)
    static constexpr int kBoxes = D / kLine;
    static constexpr int kSlot = 32 * D;               // K and V of 16 keys
    static constexpr int kStages = D == 64 ? 4 : 3;
    static constexpr int kRing = kWarpsA * kStages * kSlot;
    static constexpr int kPad = 4;
    static constexpr int kMerge = kWarpsA * kMostRows * (D + kPad) * 4;
    static constexpr int kBig = kRing > kMerge ? kRing : kMerge;
    static constexpr int kOffScale = kBig > 33024 ? kBig : 33024;             // two scales a lane and stage
    static constexpr int kOffBar = kOffScale + kWarpsA * kStages * 256;
    static constexpr int kSmem = kOffBar + kWarpsA * kStages * 8 + 1024;      // and room to begin on 1024
    static_assert(kOffScale >= 4 * (HXQ_ATTENTION_MAX_REQUESTS + 1), "room for the scan");
};

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

__device__ __forceinline__ uint32_t turn8x8(uint32_t v)
{
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

// CTAs an SM: as many as the accumulators' registers allow.
__host__ __device__ constexpr uint32_t ctas_per_sm(uint32_t D, bool few) { return D == 256 ? 2u : D == 128 && !few ? 3u : 4u; }

template <int D, int FMT, typename QT, int NT>
__global__ void __launch_bounds__(kThreadsA, ctas_per_sm(D, NT == 1)) attn_mma_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
{
    using G = Geo<D>;
    constexpr int kRows = 8 * NT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (pipe::smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ RangeShared<kWarpsA> sh;
    __shared__ float sh_m[kWarpsA][kRows], sh_l[kWarpsA][kRows];
    __shared__ uint32_t gave_up;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    let_next_start();
    if (tid == 0) {
        a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
        gave_up = 0;
    }
    Range range;
    if (!find_range<kWarpsA, kRows, kGran, kFixed>(a, sh, reinterpret_cast<uint32_t *>(smem), true, range)) return;
    __syncthreads();   // the sums in front of the requests are read: the ring may be filled

    const uint32_t ring = pipe::smem_u32(smem) + warp * (G::kStages * G::kSlot);
    const uint32_t scales = pipe::smem_u32(smem) + G::kOffScale + warp * (G::kStages * 256) + lane * 8;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + G::kOffBar) + warp * G::kStages;
    float *merge = reinterpret_cast<float *>(smem);
    if (lane == 0) {
        for (int s = 0; s < G::kStages; ++s) pipe::mbar_init(full + s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    uint32_t phase = 0;   // bit s: parity of stage s's next arrival
    // This lane's 16 bytes of key g (key g + 8: 8 rows on), and of dimensions
    // 16 g .. of keys 2 q and 2 q + 1; a row's 16-byte pieces are swapped by
    // the row's number (128-byte rows: row & 7, 64-byte rows: row / 2 & 3)
    uint32_t k_at[2], v_at[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t row = 2 * q + i;
        if (D == 64) {
            k_at[i] = g * 64 + ((q ^ (g >> 1 & 3u)) << 4);
            v_at[i] = row * 64 + (((g >> 1) ^ (row >> 1 & 3u)) << 4) + (g & 1u) * 8;
        } else {
            k_at[i] = g * 128 + (((2 * q + i) ^ g) << 4);
            v_at[i] = row * 128 + ((g ^ (row & 7u)) << 4);
        }
    }
    bool in_time = true;

    Segment seg;
    while (next_segment<kRows, kGran, kFixed>(a, range, seg)) {
        const Req &r = seg.r;
        const uint32_t h = seg.h, take = seg.take, lo = seg.lo, hi = seg.hi, r0 = seg.r0, r1 = seg.r1;
        const uint32_t key0 = seg.key0 + warp * 16;   // this warp's first 16 keys
        const int32_t before = (int32_t)r.len - (int32_t)r.n;
        auto position = [&](uint32_t row) { return a.causal ? before + (int32_t)token_of(a, row) : (int32_t)r.len - 1; };
        // a row sees keys above its floor: its position less the window, -1 without one
        auto key_floor = [&](int32_t at) { return a.window ? (int32_t)max((int64_t)at - (int64_t)a.window, (int64_t)-1) : -1; };

        // ---- the first copies: K and V of the first steps
        uint32_t valid = 0;   // bit s: the step in stage s has a block inside the cache
        const int32_t *table = a.table + (size_t)seg.b * a.width;
        auto entry = [&](uint32_t j) -> int32_t {
            const uint32_t key = key0 + j * kGran;
            uint32_t slot;
            return j < take && key < hi && key + 16 > lo ? __ldg(table + block_of(a, key, slot)) : -1;
        };
        auto issue = [&](uint32_t j, uint32_t stage, int32_t blk) {
            const uint32_t key = key0 + j * kGran;
            const bool wanted = j < take && key < hi && key + 16 > lo, ok = wanted && (uint32_t)blk < a.n_blocks;
            if (wanted && !ok && lane == 0) flag(a.status, HXQ_SERVING_BAD_BLOCK);
            valid = ok ? valid | 1u << stage : valid & ~(1u << stage);
            if (ok) {
                uint32_t slot;
                block_of(a, key, slot);
                const uint32_t bh = (uint32_t)blk * a.H + h;
                cp4(scales + stage * 256, a.ks + bh);
                cp4(scales + stage * 256 + 4, a.vs + bh);
                // the stage's last reads come before the copy
                pipe::async_proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    const int32_t row = (int32_t)(bh * a.P + slot);
                    uint8_t *dst = smem + (size_t)(warp * G::kStages + stage) * G::kSlot;
                    pipe::mbar_expect_tx(full + stage, G::kSlot);
#pragma unroll
                    for (int b = 0; b < G::kBoxes; ++b) {
                        pipe::tma_load_2d(dst + b * 2048, &kmap, full + stage, b * 128, row);
                        pipe::tma_load_2d(dst + 16 * D + b * 2048, &vmap, full + stage, b * 128, row);
                    }
                }
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

        // ---- Q: rows g + 8 n, in the order in which codes arrive
        uint32_t qf[NT][D / 16][2];
        float fac[NT][2];           // of rows 2 q and 2 q + 1, as the scores have them
        int32_t pos[NT][2], floors[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t row = r0 + g + 8 * n;
            const bool in = row < r1;
            const uint32_t tok = in ? token_of(a, row) : 0, head = h * a.G + (in ? row - tok * a.G : 0);
            const QT *p = static_cast<const QT *>(a.q) + (int64_t)(r.q0 + tok) * a.q_st + (int64_t)head * a.q_sh;
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < G::kKC; ++c)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t d0 = D == 64 ? q * 16 : (c >> 1) * 128 + (2 * q + (c & 1)) * 16;
                    const uint4 v = in ? __ldg(reinterpret_cast<const uint4 *>(p + d0) + w) : make_uint4(0, 0, 0, 0);
                    qf[n][c * 4 + w * 2][0] = v.x;
                    qf[n][c * 4 + w * 2][1] = v.y;
                    qf[n][c * 4 + w * 2 + 1][0] = v.z;
                    qf[n][c * 4 + w * 2 + 1][1] = v.w;
                }
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const QT *e = reinterpret_cast<const QT *>(&qf[n][s][w]);
                    top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[0]))));
                    top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[1]))));
                }
            top = max(top, __shfl_xor_sync(~0u, top, 1));
            top = max(top, __shfl_xor_sync(~0u, top, 2));
            // 2^(14 - exponent of the largest): into [2^14, 2^15) (below 2^-112: as far as a factor of 2^126 goes);
            // 0 and non-finite rows as they are
            const int32_t e = (int32_t)(top >> 23) - 127;
            const int32_t shift = (top == 0 || e == 128) ? 0 : max(-113, min(126, 14 - e));
            const float m = __uint_as_float((uint32_t)(127 + shift) << 23);
            const float f = a.scale_log2 * __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int w = 0; w < 2; ++w) qf[n][s][w] = to_f16x2<QT>(qf[n][s][w], m);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fac[n][i] = __shfl_sync(~0u, f, (2 * q + i) * 4);
                const uint32_t rw = r0 + 8 * n + 2 * q + i;
                pos[n][i] = rw < r1 ? position(rw) : -1;
                floors[n][i] = key_floor(pos[n][i]);
            }
        }
        const int32_t pos_first = position(r0), floor_last = key_floor(position(r1 - 1));

        // ---- key loop
        float o[D / 16][NT][4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[n][i] = -INFINITY;
                l[n][i] = 0.0f;
            }
        uint32_t stage = 0;
        for (uint32_t j = 0; j < take; ++j) {
            cp_wait<G::kStages - 2>();
            const bool live = valid >> stage & 1u;
            if (live) {
                in_time = __all_sync(~0u, bounded_wait(full + stage, phase >> stage & 1u, &gave_up, a) && a.wait_cycles);
                if (!in_time) break;
                phase ^= 1u << stage;
            }
            {
                const uint32_t into = stage == 0 ? G::kStages - 1 : stage - 1;
                issue(j + G::kStages - 1, into, next);
                next = entry(j + G::kStages);
            }
            if (live) {
                const uint32_t src = ring + stage * G::kSlot;
                const uint2 sc = pipe::lds64(scales + stage * 256);
                float s[NT][4], s2[NT][4];   // two chains of products
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.0f;
#pragma unroll
                for (int c = 0; c < G::kKC; ++c) {
                    const uint32_t at = src + (c >> 1) * 2048 + k_at[c & 1];
                    const uint4 ka = pipe::lds128(at), kb = pipe::lds128(at + 8 * G::kLine);   // keys g, g + 8
                    const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        codes_to_f16<FMT>(wa[i], a0, a2);
                        codes_to_f16<FMT>(wb[i], a1, a3);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            pipe::mma16816_f16(i & 1 ? s2[n] : s[n], a0, a1, a2, a3, qf[n][c * 4 + i][0], qf[n][c * 4 + i][1]);
                    }
                }
                const uint32_t key = key0 + j * kGran;
                float lv, inv;
                bool zero;
                value_scale(__uint_as_float(sc.y), lv, inv, zero);
                const float ks = __uint_as_float(sc.x);
                // scores: [0], [1] of key g and rows 2 q, 2 q + 1; [2], [3] of key g + 8
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e] + s2[n][e], fac[n][e & 1] * ks, lv);
                if (!((int32_t)(key + 15) <= pos_first && (int32_t)key > floor_last)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int32_t kp = (int32_t)(key + g + (e >> 1) * 8);
                            if (kp > pos[n][e & 1] || kp <= floors[n][e & 1]) s[n][e] = -INFINITY;
                        }
                }
                bool raise = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) raise |= fmaxf(s[n][i], s[n][i + 2]) > m[n][i] + kRaiseA;
                if (__any_sync(~0u, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float al[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float top = fmaxf(s[n][i], s[n][i + 2]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                            const float to = fmaxf(m[n][i], top);
                            al[i] = to == -INFINITY ? 1.0f : ex2(m[n][i] - to);
                            m[n][i] = to;
                            l[n][i] *= al[i];
                        }
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            o[i][n][0] *= al[0];
                            o[i][n][1] *= al[1];
                            o[i][n][2] *= al[0];
                            o[i][n][3] *= al[1];
                        }
                    }
                }
                uint32_t p[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float ms = (m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1]) - kLift;
                        w[e] = ex2(s[n][e] - ms);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // a row that sees none of the keys takes nothing from their block, whatever its scale
                        const float sum = w[i] + w[i + 2];
                        l[n][i] += sum == 0.0f ? 0.0f : sum * inv;
                        const __half2 hh = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
                        const uint32_t v = turn8x8(*reinterpret_cast<const uint32_t *>(&hh));
                        p[n][i] = zero ? 0u : v;
                    }
                }
                const bool tail = key + 16 > hi || key < lo;
#pragma unroll
                for (int c = 0; c < G::kVC; ++c) {
                    uint32_t vw[4][4];
#pragma unroll
                    for (int ts = 0; ts < 4; ++ts) {
                        if (G::kVB == 16) {
                            const uint4 v = pipe::lds128(src + 16 * D + c * 2048 + (ts >> 1) * 8 * G::kLine + v_at[ts & 1]);
                            vw[ts][0] = v.x;
                            vw[ts][1] = v.y;
                            vw[ts][2] = v.z;
                            vw[ts][3] = v.w;
                        } else {
                            const uint2 v = pipe::lds64(src + 16 * D + (ts >> 1) * 8 * G::kLine + v_at[ts & 1]);
                            vw[ts][0] = v.x;
                            vw[ts][1] = v.y;
                            vw[ts][2] = vw[ts][3] = 0;
                        }
                    }
                    if (tail) {
                        // slots behind the last key and in front of the first may hold anything
#pragma unroll
                        for (int ts = 0; ts < 4; ++ts)
                            if (key + 2 * q + (ts & 1) + (ts >> 1) * 8 - lo >= hi - lo) vw[ts][0] = vw[ts][1] = vw[ts][2] = vw[ts][3] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < G::kVB / 4; ++i)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            // bytes 2 half, 2 half + 1 of two keys: (a, b, a, b); two dimensions of the tile's 16
                            const uint32_t sel = half ? 0x7362 : 0x5140;
                            uint32_t a0, a1, a2, a3;
                            codes_to_f16<FMT>(__byte_perm(vw[0][i], vw[1][i], sel), a0, a1);
                            codes_to_f16<FMT>(__byte_perm(vw[2][i], vw[3][i], sel), a2, a3);
                            const int t = c * (G::kVB / 2) + i * 2 + half;
#pragma unroll
                            for (int n = 0; n < NT; ++n) pipe::mma16816_f16(o[t][n], a0, a1, a2, a3, p[n][0], p[n][1]);
                        }
                }
            }
            stage = stage == G::kStages - 1 ? 0 : stage + 1;
        }
        cp_wait<0>();

        // ---- join the four warps
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(~0u, l[n][i], d);
                if (g == 0) {
                    sh_m[warp][8 * n + 2 * q + i] = m[n][i];
                    sh_l[warp][8 * n + 2 * q + i] = l[n][i];
                }
            }
        in_time = __syncthreads_and(in_time);   // all four warps go on, or none
        if (!in_time) break;
        float *mine = merge + warp * kRows * (D + G::kPad);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t rr = 8 * n + 2 * q + i;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarpsA; ++w) top = fmaxf(top, sh_m[w][rr]);
                const float wt = top == -INFINITY ? 1.0f : ex2(m[n][i] - top);
#pragma unroll
                for (int c = 0; c < G::kVC; ++c)
#pragma unroll
                    for (int t = 0; t < G::kVB / 2; t += 2) {
                        const float(&x)[4] = o[c * (G::kVB / 2) + t][n], (&y)[4] = o[c * (G::kVB / 2) + t + 1][n];
                        *reinterpret_cast<float4 *>(mine + rr * (D + G::kPad) + c * 128 + g * G::kVB + 2 * t) =
                            make_float4(x[i] * wt, x[i + 2] * wt, y[i] * wt, y[i + 2] * wt);
                    }
            }
        __syncthreads();
        const bool whole = seg.begins && take == seg.n;
        float *part = a.part + (size_t)(2 * blockIdx.x + (seg.begins ? 1 : 0)) * part_floats<kMostRows, D>();
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
                    a.lse[(size_t)tok * a.Hq + head] = sum == 0.0f ? -INFINITY : (top - kLift + log2f(sum)) * 0.69314718055994531f;
            } else {
                *reinterpret_cast<float4 *>(part + rr * D + d) = v;
                if (d == 0) {
                    part[kMostRows * D + rr] = top;
                    part[kMostRows * D + kMostRows + rr] = sum;
                }
            }
        }
        if (seg.begins && take < seg.n && tid == 0) a.desc[blockIdx.x] = cut_unit(range, seg);
        pipe::async_proxy_fence();
        __syncthreads();   // the ring is free again
    }
    if (!in_time) {
        if (lane == 0) flag(a.status, HXQ_SERVING_TIMEOUT);
        let_copies_end();
    }
}

template <int D, typename QT, int NT> __global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs a)
{
    wait_previous();
    join_row<8 * NT, kMostRows, D, D == 256 ? 4 : 8, QT>(a, a.desc, a.part, blockIdx.x, blockIdx.y * 4 + (threadIdx.x >> 5));
}

// The codes as rows of D bytes, in boxes of 16 rows of 128 (64) bytes.
bool encode_codes(CUtensorMap *map, const uint8_t *codes, const AttnArgs &a, uint32_t D)
{
    const pipe::EncodeTiledFn enc = pipe::encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {D, (cuuint64_t)a.n_blocks * a.H * a.P}, strides[1] = {D};
    const cuuint32_t box[2] = {D >= 128 ? 128u : 64u, 16u}, step[2] = {1u, 1u};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, D >= 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The same for both kernels' cut units: first those of this file's kernel.
template <int D, typename QT>
__global__ void __launch_bounds__(128) attn_join_both_kernel(const __grid_constant__ AttnArgs a, const int4 *tc_desc, const float *tc_part, uint32_t few)
{
    wait_previous();
    const uint32_t warp = threadIdx.x >> 5;
    if (blockIdx.x < few) join_row<16, kMostRows, D, 4, QT>(a, a.desc, a.part, blockIdx.x >> 2, (blockIdx.x & 3u) * 4 + warp);
    else {
        const uint32_t i = blockIdx.x - few;
        join_row<kTcRows, kTcRows, D, 4, QT>(a, tc_desc, tc_part, i / (kTcRows / 4), i % (kTcRows / 4) * 4 + warp);
    }
}

template <int D, int FMT, typename QT, int NT> cudaError_t launch_one(const AttnArgs &a, const AttnArgs *tc, uint32_t grid, uint32_t tc_grid, cudaStream_t s)
{
    auto kernel = attn_mma_kernel<D, FMT, QT, NT>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(kernel, Geo<D>::kSmem, ready);
    if (e != cudaSuccess) return e;
    CUtensorMap kmap, vmap;
    if (!encode_codes(&kmap, a.k, a, D) || !encode_codes(&vmap, a.v, a, D)) return cudaErrorInvalidValue;
    kernel<<<grid, kThreadsA, Geo<D>::kSmem, s>>>(a, kmap, vmap);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if constexpr (D != 256 && NT == 2) {
        if (tc) {
            // beside each other: the kernel for many rows starts with this one
            if ((e = launch_attn_tc(*tc, D, FMT, std::is_same<QT, __half>::value ? HXQ_ELEM_F16 : HXQ_ELEM_BF16, tc_grid, s)) != cudaSuccess) return e;
            AttnArgs both = a;
            both.row_min = 0;
            both.row_max = 0xffffffffu;
            return launch_behind(attn_join_both_kernel<D, QT>, dim3(grid * 4 + tc_grid * (kTcRows / 4)), dim3(128), 0, s, both,
                                 (const int4 *)tc->desc, (const float *)tc->part, grid * 4);
        }
    }
    return launch_behind(attn_join_kernel<D, QT, NT>, dim3(grid, 2 * NT), dim3(128), 0, s, a);
}

template <int D, int FMT, typename QT> cudaError_t launch_rows(const AttnArgs &a, const AttnArgs *tc, bool few, uint32_t grid, uint32_t tc_grid, cudaStream_t s)
{
    if constexpr (D == 256) return launch_one<D, FMT, QT, 1>(a, nullptr, grid, 0, s);   // 16 rows' accumulators would not fit
    else return few ? launch_one<D, FMT, QT, 1>(a, nullptr, grid, 0, s) : launch_one<D, FMT, QT, 2>(a, tc, grid, tc_grid, s);
}

template <int D> cudaError_t launch_dim(const AttnArgs &a, const AttnArgs *tc, uint32_t fmt, int elem, bool few, uint32_t grid, uint32_t tc_grid, cudaStream_t s)
{
    if (elem == HXQ_ELEM_BF16)
        return fmt == HXQ_KV_INT8 ? launch_rows<D, HXQ_KV_INT8, __nv_bfloat16>(a, tc, few, grid, tc_grid, s)
                                  : launch_rows<D, HXQ_KV_E4M3, __nv_bfloat16>(a, tc, few, grid, tc_grid, s);
    return fmt == HXQ_KV_INT8 ? launch_rows<D, HXQ_KV_INT8, __half>(a, tc, few, grid, tc_grid, s)
                              : launch_rows<D, HXQ_KV_E4M3, __half>(a, tc, few, grid, tc_grid, s);
}

cudaError_t launch_attn_mma(const AttnArgs &a, const AttnArgs *tc, uint32_t D, uint32_t fmt, int elem, bool few, uint32_t grid, uint32_t tc_grid,
                            cudaStream_t s)
{
    return D == 64 ? launch_dim<64>(a, tc, fmt, elem, few, grid, tc_grid, s)
                   : D == 128 ? launch_dim<128>(a, tc, fmt, elem, few, grid, tc_grid, s) : launch_dim<256>(a, tc, fmt, elem, few, grid, tc_grid, s);
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
    if ((uint64_t)c->n_blocks * c->block_tokens * c->n_heads >= (1ull << 31)) return HXQ_ERR_INVALID_ARG;   // rows of a copy's map
    if (p->window && !p->causal) return HXQ_ERR_INVALID_ARG;
    if (!(p->scale >= 0.0f) || p->scale > 3.402823466e38f) return HXQ_ERR_INVALID_ARG;
    return HXQ_OK;
}

// Workspace: a word group for every CTA, then the partial results, of this
// kernel and of the one for many rows.
struct AttnLayout {
    uint32_t ctas, tc_ctas;
    bool few;                     // tiles of 8 rows
    size_t part, tc_desc, tc_part, bytes;
};

// What a wait inside a kernel may take: about a second.
std::atomic<uint32_t> wait_cycles{2000000000u};

// Requests with more rows than this go to the tcgen05 kernel.  16 requests of
// 4096 keys, 8 heads, int8, rows of a request: us a call here (tiles of 16) and
// there: heads of 128, 32: 87, 105; 48: 120, 105; 64: 153, 107; 96: 214, 107;
// heads of 64: 65, 89; 87, 89; 109, 87; 155, 89.  (They meet at about 40 and 48.)
constexpr uint32_t kFewRows = 64;

AttnLayout attn_layout(uint32_t D, uint64_t most_rows)   // most_rows: of a request, as the caller says
{
    AttnLayout l;
    const uint32_t sms = (uint32_t)sm_count();
    // tiles of 8 rows or of 16, the same keys: 8 rows 44 and 52 us (heads of 64: 35, 40), 12 rows 69 and 54 (52, 42)
    l.few = D == 256 || most_rows <= 8;
    l.ctas = sms * ctas_per_sm(D, l.few);
    l.tc_ctas = D != 256 && most_rows > kFewRows ? sms : 0;
    l.part = l.ctas * sizeof(int4);
    l.tc_desc = l.part + (size_t)l.ctas * 2 * (kMostRows * D + 2 * kMostRows) * sizeof(float);
    l.tc_part = l.tc_desc + l.tc_ctas * sizeof(int4);
    l.bytes = l.tc_part + (size_t)l.tc_ctas * 2 * (kTcRows * D + 2 * kTcRows) * sizeof(float);
    return l;
}

}  // namespace serving
}  // namespace hxq

using namespace hxq::serving;

extern "C" {

// Not part of the API: lets a test see the waits of the attention kernels run
// out. Returns the limit there was.
uint32_t hxq_serving_wait_cycles(uint32_t cycles) { return wait_cycles.exchange(cycles); }

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
    const Runs out = {(uintptr_t)args->d_out, {args->n_rows, args->n_heads}, {args->out_stride_t, args->out_stride_h}, cache->head_dim, 2},
               q = {(uintptr_t)args->d_q, {args->n_rows, args->n_heads}, {args->q_stride_t, args->q_stride_h}, cache->head_dim, 2};
    if (!out.apart() || !out.may_overwrite(q)) return HXQ_ERR_INVALID_ARG;
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
    a.wait_cycles = wait_cycles.load(std::memory_order_relaxed);
    a.scale_log2 = args->scale * 1.4426950408889634f;
    uint8_t *ws = static_cast<uint8_t *>(d_workspace);
    a.desc = reinterpret_cast<int4 *>(ws);
    a.part = reinterpret_cast<float *>(ws + lay.part);
    // Few rows of a request: this file's kernel. More: the tcgen05 kernel.
    // Without rows of the other kind a launch ends after its scan of the
    // lengths.
    AttnArgs tc = a;
    if (lay.tc_ctas) {
        a.row_max = kFewRows;
        tc.row_min = kFewRows;
        tc.desc = reinterpret_cast<int4 *>(ws + lay.tc_desc);
        tc.part = reinterpret_cast<float *>(ws + lay.tc_part);
    }
    const cudaError_t e = launch_attn_mma(a, lay.tc_ctas ? &tc : nullptr, cache->head_dim, cache->format, args->elem, lay.few, lay.ctas,
                                          lay.tc_ctas, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return HXQ_ERR_CUDA;
    }
    return launched(lay.tc_ctas ? 3 : 2);
}

}  // extern "C"
