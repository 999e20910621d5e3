// kv_prefill.cu -- attention over the 8-bit cache for many query rows per
// key (prompts, chunks of prompts) on tcgen05.
//
// The mathematics is kv_attention.cu's: products on codes alone, block scales
// inside the exponent and the row sums.  A CTA takes 256 rows (tokens x heads
// of a group) of one (request, cache head), two tiles of 128, against 128 keys
// at a time:
//   warps 0-7   one row per thread (tile = warp / 4): Q scaled into f16 and
//               into shared memory once, then for every 128 keys the scores
//               out of tensor memory, exp2, weights back into tensor memory
//               as f16 over the scores' columns; at the end the row out;
//   warps 8-11  codes: global memory -> registers (one step ahead) -> f16 ->
//               shared memory, keys [key][dim] and values transposed
//               [dim][key], both K-major with 128-byte swizzle; the block
//               scales of every 16 keys;
//   warp 12     one thread issues S = Q K^T (both operands in shared memory)
//               and O += P V (P in tensor memory).
// The two tiles take turns: while one is at its exponentials, the tensor
// cores work for the other.  Tensor memory: S/P of tile t at column 128 t,
// O of tile t at 256 + 128 t, all 512 columns, one CTA an SM.
//
// The running maximum is lazy: weights are taken against the maximum so far
// and only where one would pass 2^8 (f16 holds 2^16) is it raised and O
// rescaled, which after the first keys is rare, so that the rescale needs no
// warps of its own and the scores are read from tensor memory once.
//
// Work is cut and joined as in kv_attention.cu, with granules of 128 keys.
// Every wait is bounded; one that runs out is recorded and the CTA unwinds.
#include "kv_attention.cuh"

#include "tc_pipe.cuh"

namespace hxq {
namespace serving {

constexpr int kKeys = 128;                 // keys of a step
constexpr int kTile = 128;                 // rows of a tile
constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kWarpsT = kSoftWarps + kConvWarps + 1;
constexpr int kThreadsT = kWarpsT * 32;
constexpr int kScaleSlots = 4;
constexpr float kRaise = 8.0f;             // log2 of the largest weight before the maximum is raised

template <int D> struct TcGeo {
    static constexpr int kQ = kTile * D * 2;           // bytes of a tile of Q
    static constexpr int kK = kKeys * D * 2;           // of a step's keys, and of its values
    static constexpr int kOffK = 2 * kQ, kOffV = kOffK + 2 * kK, kOffS = kOffV + 2 * kK;
    static constexpr int kOffBar = kOffS + kScaleSlots * 8 * 16;
    static constexpr int kSmem = kOffBar + 256 + 1024;
    static constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
    static constexpr uint32_t kIdescPV = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
};

// K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

__device__ __forceinline__ void tc_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(pipe::smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t *v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct Bars {
    uint64_t q_full[2], s_full[2], p_full[2], o_done[2], k_full[2], k_empty[2], v_full[2], v_empty[2], drained;
    uint32_t tmem, abort;
};

// Bounded wait; false once it, or another one of the CTA, has run out.
struct Waiter {
    Bars *bars;
    uint32_t *status;
    __device__ __forceinline__ bool operator()(uint64_t *bar, uint32_t parity) const
    {
        if (pipe::mbar_try(bar, parity)) return true;
        const uint64_t t0 = clock64();
        while (!pipe::mbar_try(bar, parity)) {
            if (*(volatile uint32_t *)&bars->abort) return false;
            if (clock64() - t0 > pipe::kWaitCycles) {
                *(volatile uint32_t *)&bars->abort = 1u;
                flag(status, HXQ_SERVING_TIMEOUT);
                return false;
            }
        }
        return true;
    }
};

// A step of 128 keys within the CTA's range, for the converters, which run
// ahead of the other warps.
struct Cursor {
    Range range;
    Segment seg;
    uint32_t j;
    bool ok;
    __device__ __forceinline__ void next(const AttnArgs &a)
    {
        if (!ok) return;
        if (++j >= seg.take) {
            ok = next_segment<kTcRows, kKeys>(a, range, seg);
            j = 0;
        }
    }
};

template <int D, int FMT, typename QT>
__global__ void __launch_bounds__(kThreadsT, 1) attn_tc_kernel(const __grid_constant__ AttnArgs a)
{
    using G = TcGeo<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (pipe::smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ RangeShared<kWarpsT> sh;
    Bars *bars = reinterpret_cast<Bars *>(smem + G::kOffBar);
    float4 *scales = reinterpret_cast<float4 *>(smem + G::kOffS);   // [slot][16-key group]: ks, log2 vs, 1 / vs
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = pipe::smem_u32(smem);

    if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    Range range;
    if (!find_range<kWarpsT, kTcRows, kKeys>(a, sh, false, range)) return;
    if (tid == 0) {
        for (int t = 0; t < 2; ++t) {
            pipe::mbar_init(&bars->q_full[t], kTile);
            pipe::mbar_init(&bars->s_full[t], 1);
            pipe::mbar_init(&bars->p_full[t], kTile);
            pipe::mbar_init(&bars->o_done[t], 1);
            pipe::mbar_init(&bars->k_full[t], kConvWarps * 32);
            pipe::mbar_init(&bars->k_empty[t], 1);
            pipe::mbar_init(&bars->v_full[t], kConvWarps * 32);
            pipe::mbar_init(&bars->v_empty[t], 1);
        }
        pipe::mbar_init(&bars->drained, 1);
        bars->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpsT - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pipe::smem_u32(&bars->tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bars->tmem;
    const Waiter wait{bars, a.status};

    if (warp < kSoftWarps) {
        // ------------------------------------------------------- rows
        const uint32_t t = warp >> 2, rr = tid & (kTile - 1);          // tile, row of it
        const uint32_t lanes = (warp & 3u) << 21;                      // this warp's 32 lanes of tensor memory
        const uint32_t tS = tmem + lanes + t * 128u, tO = tmem + lanes + 256u + t * 128u;
        uint32_t n_q = 0, n_s = 0;                                     // Q tiles and steps so far
        uint32_t step0 = 0;                                            // CTA's steps before this segment
        Segment seg;
        bool ok = true;
        while (ok && next_segment<kTcRows, kKeys>(a, range, seg)) {
            const Req &r = seg.r;
            if (t == 1 && seg.r1 - seg.r0 <= (uint32_t)kTile) {
                step0 += seg.take;
                continue;
            }
            const uint32_t tr0 = seg.r0 + t * kTile, tr1 = min(tr0 + kTile, seg.r1), row = tr0 + rr;
            const bool in = row < tr1;
            const int32_t before = (int32_t)((int64_t)r.len - r.n);
            auto position = [&](uint32_t rw) { return a.causal ? before + (int32_t)(rw / a.G) : (int32_t)r.len - 1; };
            auto key_floor = [&](int32_t at) { return a.window ? (int32_t)max((int64_t)at - (int64_t)a.window, (int64_t)-1) : -1; };
            const int32_t pos_first = position(tr0), pos_last = position(tr1 - 1), pos = in ? position(row) : pos_last;
            const int32_t floor_last = key_floor(pos_last), floor = key_floor(pos);
            const uint32_t tok = r.q0 + (in ? row / a.G : 0), head = seg.h * a.G + (in ? row % a.G : 0);
            float fac;
            {
                // Q: the row's largest into [2^14, 2^15), 0 and non-finite rows as they are
                const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const QT *>(a.q) + (int64_t)tok * a.q_st + (int64_t)head * a.q_sh);
                uint4 v[D / 8];
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    v[c] = in ? __ldg(p + c) : make_uint4(0, 0, 0, 0);
                    const QT *e = reinterpret_cast<const QT *>(&v[c]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[i]))));
                }
                const int32_t e2 = (int32_t)(top >> 23) - 127;
                const int32_t shift = (top == 0 || e2 == 128) ? 0 : max(-100, min(100, 14 - e2));
                const float m = __uint_as_float((uint32_t)(127 + shift) << 23);
                fac = a.scale_log2 * __uint_as_float((uint32_t)(127 - shift) << 23);
                const uint32_t dst = base + t * G::kQ + rr * 128u;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const QT *e = reinterpret_cast<const QT *>(&v[c]);
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __half2 h = __floats2half2_rn(Elem<QT>::to(e[2 * i]) * m, Elem<QT>::to(e[2 * i + 1]) * m);
                        w[i] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    sts128(dst + (c >> 3) * (kTile * 128u) + (((c & 7) ^ (rr & 7)) << 4), w[0], w[1], w[2], w[3]);
                }
                pipe::async_proxy_fence();
                pipe::mbar_arrive(&bars->q_full[t]);
                ++n_q;
            }
            float M = -INFINITY, l = 0.0f;
            for (uint32_t j = 0; j < seg.take; ++j) {
                const uint32_t key0 = (seg.first + seg.rem + j) * kKeys;
                ok = __all_sync(~0u, wait(&bars->s_full[t], n_s & 1u));
                if (!ok) break;
                fence_after();
                const float4 *sc = scales + ((step0 + j) & (kScaleSlots - 1)) * 8;
                const bool all = (int32_t)(key0 + kKeys - 1) <= pos_first && (int32_t)key0 > floor_last;
                uint32_t p[kKeys / 2];
                float add = 0.0f, top = -INFINITY;
                const bool begin = __any_sync(~0u, M == -INFINITY);
                // weights against the maximum so far; only the largest score
                // while some row has none yet
                auto pass = [&](bool only_top) {
                    const float ms = M == -INFINITY ? 0.0f : M;
                    add = 0.0f;
                    top = -INFINITY;
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        uint32_t s[32];
                        tm_ld32(tS + c * 32, s);
                        wait_ld();
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float4 b = sc[c * 2 + g];
                            const float f = fac * b.x, off = b.y - ms;
                            float sum = 0.0f;
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float t0 = fmaf(__uint_as_float(s[g * 16 + i]), f, off);
                                float t1 = fmaf(__uint_as_float(s[g * 16 + i + 1]), f, off);
                                if (!all) {
                                    const int32_t k = (int32_t)(key0 + c * 32 + g * 16 + i);
                                    if (k > pos || k <= floor) t0 = -INFINITY;
                                    if (k + 1 > pos || k + 1 <= floor) t1 = -INFINITY;
                                }
                                top = fmaxf(top, fmaxf(t0, t1));
                                if (!only_top) {
                                    const float w0 = ex2(t0), w1 = ex2(t1);
                                    sum += w0 + w1;
                                    const __half2 h = __floats2half2_rn(w0, w1);
                                    p[(c * 32 + g * 16 + i) / 2] = *reinterpret_cast<const uint32_t *>(&h);
                                }
                            }
                            // a row that sees none of the 16 keys takes nothing from their block, whatever its scale
                            add += sum == 0.0f ? 0.0f : sum * b.z;
                        }
                    }
                };
                // raise the maximum to the largest score seen
                auto raise = [&]() {
                    const float to = fmaxf(M, top == -INFINITY ? M : top + (M == -INFINITY ? 0.0f : M));
                    const float al = to == -INFINITY ? 1.0f : ex2(M - to);
                    M = to;
                    l *= al;
                    if (j > 0) {
                        ok = __all_sync(~0u, wait(&bars->o_done[t], (n_s - 1) & 1u));
                        if (!ok) return;
                        fence_after();
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tm_ld32(tO + c * 32, o);
                            wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                            tm_st32(tO + c * 32, o);
                        }
                        wait_st();
                    }
                };
                if (begin) {
                    pass(true);
                    raise();
                    if (!ok) break;
                }
                pass(false);
                if (__any_sync(~0u, top > kRaise)) {
                    raise();
                    if (!ok) break;
                    pass(false);
                }
                l += add;
                tm_st32(tS, p);
                tm_st32(tS + 32, p + 32);
                wait_st();
                fence_before();
                pipe::mbar_arrive(&bars->p_full[t]);
                ++n_s;
            }
            if (!ok) break;
            step0 += seg.take;
            ok = __all_sync(~0u, wait(&bars->o_done[t], (n_s - 1) & 1u));
            if (!ok) break;
            fence_after();
            const bool whole = seg.rem == 0 && seg.take == seg.n;
            if (whole) {
                const float f = l == 0.0f ? 0.0f : 1.0f / l;
                QT *dst = static_cast<QT *>(a.out) + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh;
                const bool wide = (((uintptr_t)dst) & 15u) == 0;
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tm_ld32(tO + c * 32, o);
                    wait_ld();
                    if (in) {
                        QT e[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) e[i] = Elem<QT>::from(__uint_as_float(o[i]) * f);
                        if (wide) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) reinterpret_cast<uint4 *>(dst + c * 32)[i] = reinterpret_cast<const uint4 *>(e)[i];
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) dst[c * 32 + i] = e[i];
                        }
                    }
                }
                if (in && a.lse)
                    a.lse[(size_t)tok * a.Hq + head] = l == 0.0f ? -INFINITY : (M + log2f(l)) * 0.69314718055994531f;
            } else {
                float *part = a.part + (size_t)(2 * blockIdx.x + (seg.rem == 0 ? 1 : 0)) * part_floats<kTcRows, D>();
                const uint32_t pr = t * kTile + rr;
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tm_ld32(tO + c * 32, o);
                    wait_ld();
                    if (in) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            reinterpret_cast<uint4 *>(part + (size_t)pr * D + c * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
                if (in) {
                    part[kTcRows * D + pr] = M;
                    part[kTcRows * D + kTcRows + pr] = l;
                }
                if (seg.rem == 0 && tid == 0) a.desc[blockIdx.x] = cut_unit(range, seg);
            }
            fence_before();   // O is read before the next segment's products, which wait for its weights
        }
    } else if (warp < kSoftWarps + kConvWarps) {
        // ------------------------------------------------------- codes
        const uint32_t ct = tid - kSoftWarps * 32, cw = ct >> 5;
        constexpr int kLanesK = D / 16;                       // lanes of a key row (16 codes each)
        constexpr int kNK = kKeys * kLanesK / 128;            // key loads of a thread: 8 or 4
        constexpr int kLanesV = D / 4;                        // lanes of a value row (4 codes each)
        constexpr int kNV = 16 * kLanesV / 128;               // groups of 8 value rows of a thread: 4 or 2
        const uint32_t kc = lane % kLanesK, kr = cw * (32 / kLanesK) + lane / kLanesK;   // K: piece, row of every load
        const uint32_t vd = (lane % kLanesV) * 4, vg = cw * (32 / kLanesV) + lane / kLanesV;   // V: first dim, group of every load
        // values: position i of a word holds dim vd + (i + turn) % 4, so that the
        // 8 lanes of a store phase write 8 different 16-byte columns
        const uint32_t turn = (lane >> 1) & 3u;
        const uint32_t k0 = turn, k1 = (turn + 1) & 3u, k2 = (turn + 2) & 3u, k3 = (turn + 3) & 3u;
        const uint32_t selA = k0 | (k0 + 4) << 4 | k1 << 8 | (k1 + 4) << 12, selB = k2 | (k2 + 4) << 4 | k3 << 8 | (k3 + 4) << 12;
        const uint32_t vdim[4] = {vd + k0, vd + k1, vd + k2, vd + k3};
        constexpr uint32_t kStepK = kKeys / kNK, kStepV = 16 / kNV;   // rows, groups between a thread's loads

        Cursor cur{range, {}, 0, true};
        cur.ok = next_segment<kTcRows, kKeys>(a, cur.range, cur.seg);
        Cursor nxt = cur;
        int32_t ek[kNK], ev[kNV], es = -1;
        uint4 kw[kNK];
        uint32_t vw[kNV][8];
        float vs_of[kNV], s_k = 0.0f, s_v = 0.0f;
        bool s_ok = false;
        // table entries of a step's rows
        auto entries = [&](const Cursor &c) {
            if (!c.ok) return;
            const uint32_t key0 = (c.seg.first + c.seg.rem + c.j) * kKeys;
            const int32_t *row = a.table + (size_t)c.seg.b * a.width;
            auto entry = [&](uint32_t key) -> int32_t { return key < c.seg.hi ? __ldg(row + key / a.P) : -1; };
#pragma unroll
            for (int i = 0; i < kNK; ++i) ek[i] = entry(key0 + i * kStepK + (kr & ~15u));
#pragma unroll
            for (int i = 0; i < kNV; ++i) ev[i] = entry(key0 + (i * kStepV + vg) * 8);
            if (ct < 8) {
                es = entry(key0 + ct * 16);
                if (key0 + ct * 16 < c.seg.hi && (uint32_t)es >= a.n_blocks) flag(a.status, HXQ_SERVING_BAD_BLOCK);
            }
        };
        auto load_k = [&](const Cursor &c) {
            if (!c.ok) return;
            const uint32_t key0 = (c.seg.first + c.seg.rem + c.j) * kKeys;
#pragma unroll
            for (int i = 0; i < kNK; ++i) {
                const uint32_t key = key0 + i * kStepK + kr;
                kw[i] = make_uint4(0, 0, 0, 0);
                if ((uint32_t)ek[i] < a.n_blocks)
                    kw[i] = __ldg(reinterpret_cast<const uint4 *>(a.k + (((size_t)(uint32_t)ek[i] * a.H + c.seg.h) * a.P + key % a.P) * D + kc * 16));
            }
            s_ok = (uint32_t)es < a.n_blocks;
            if (ct < 8 && s_ok) {
                s_k = __ldg(a.ks + (size_t)(uint32_t)es * a.H + c.seg.h);
                s_v = __ldg(a.vs + (size_t)(uint32_t)es * a.H + c.seg.h);
            }
        };
        auto load_v = [&](const Cursor &c) {
            if (!c.ok) return;
            const uint32_t key0 = (c.seg.first + c.seg.rem + c.j) * kKeys;
#pragma unroll
            for (int i = 0; i < kNV; ++i) {
                const uint32_t key = key0 + (i * kStepV + vg) * 8;
                const bool in = (uint32_t)ev[i] < a.n_blocks;
                const size_t bh = (size_t)(in ? (uint32_t)ev[i] : 0u) * a.H + c.seg.h;
                vs_of[i] = in ? __ldg(a.vs + bh) : 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    vw[i][u] = in ? __ldg(reinterpret_cast<const uint32_t *>(a.v + (bh * a.P + key % a.P + u) * D + vd)) : 0u;
            }
        };
        entries(cur);
        load_k(cur);
        load_v(cur);
        nxt.next(a);
        entries(nxt);
        bool ok = true;
        for (uint32_t it = 0; cur.ok; ++it) {
            const uint32_t st = it & 1u, par = (it >> 1) & 1u;
            const uint32_t key0 = (cur.seg.first + cur.seg.rem + cur.j) * kKeys, hi = cur.seg.hi;
            if (it >= 2) ok = __all_sync(~0u, wait(&bars->k_empty[st], par ^ 1u));
            if (!ok) break;
            const uint32_t kb = base + G::kOffK + st * G::kK;
#pragma unroll
            for (int i = 0; i < kNK; ++i) {
                const uint32_t row = i * kStepK + kr, w[4] = {kw[i].x, kw[i].y, kw[i].z, kw[i].w};
                uint32_t h[8];
#pragma unroll
                for (int u = 0; u < 4; ++u) codes_to_f16<FMT>(w[u], h[2 * u], h[2 * u + 1]);
                // 16 codes: two 16-byte columns; odd column first in the second half of a row of 128, away from the
                // first half's even ones
                const uint32_t half = kc >> 2, c0 = (kc & 3u) * 2, odd = half;
                const uint32_t dst = kb + half * (kKeys * 128u) + row * 128u;
                const uint32_t a0 = dst + (((c0 + odd) ^ (row & 7u)) << 4), a1 = dst + (((c0 + (odd ^ 1u)) ^ (row & 7u)) << 4);
                sts128(a0, odd ? h[4] : h[0], odd ? h[5] : h[1], odd ? h[6] : h[2], odd ? h[7] : h[3]);
                sts128(a1, odd ? h[0] : h[4], odd ? h[1] : h[5], odd ? h[2] : h[6], odd ? h[3] : h[7]);
            }
            if (ct < 8) {
                float4 b = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);   // keys outside: no weight
                if (s_ok) {
                    bool zero;
                    b.x = s_k;
                    value_scale(s_v, b.y, b.z, zero);
                }
                scales[(it & (kScaleSlots - 1)) * 8 + ct] = b;
            }
            pipe::async_proxy_fence();
            pipe::mbar_arrive(&bars->k_full[st]);
            load_k(nxt);
            if (it >= 2) ok = __all_sync(~0u, wait(&bars->v_empty[st], par ^ 1u));
            if (!ok) break;
            const uint32_t vb = base + G::kOffV + st * G::kK;
#pragma unroll
            for (int i = 0; i < kNV; ++i) {
                const uint32_t grp = i * kStepV + vg, key = key0 + grp * 8;
                const bool drop = vs_of[i] < 7.8886090522101181e-31f;   // blocks below 2^-100 count as 0
                if (drop || key + 8 > hi) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (drop || key + u >= hi) vw[i][u] = 0;   // slots behind the last key may hold anything
                }
                uint32_t o[4][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    codes_to_f16<FMT>(__byte_perm(vw[i][2 * u], vw[i][2 * u + 1], selA), o[0][u], o[1][u]);
                    codes_to_f16<FMT>(__byte_perm(vw[i][2 * u], vw[i][2 * u + 1], selB), o[2][u], o[3][u]);
                }
                const uint32_t dst = vb + (grp >> 3) * (D * 128u);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    sts128(dst + vdim[u] * 128u + (((grp & 7u) ^ (vdim[u] & 7u)) << 4), o[u][0], o[u][1], o[u][2], o[u][3]);
            }
            pipe::async_proxy_fence();
            pipe::mbar_arrive(&bars->v_full[st]);
            load_v(nxt);
            cur = nxt;
            nxt.next(a);
            entries(nxt);
        }
    } else if (lane == 0) {
        // ------------------------------------------------------- products
        uint32_t it = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        Segment seg;
        bool ok = true;
        auto qk = [&](uint32_t t, uint32_t st) {
            const uint32_t qa = base + t * G::kQ, kb = base + G::kOffK + st * G::kK;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
                tc_mma_ss(tmem + t * 128u, desc_sw128(qa + (kk >> 2) * (kTile * 128u) + (kk & 3) * 32u),
                          desc_sw128(kb + (kk >> 2) * (kKeys * 128u) + (kk & 3) * 32u), G::kIdescQK, kk != 0);
            tc_commit(&bars->s_full[t]);
        };
        while (ok && next_segment<kTcRows, kKeys>(a, range, seg)) {
            const uint32_t tiles = seg.r1 - seg.r0 > (uint32_t)kTile ? 2u : 1u;
            ok = wait(&bars->k_full[it & 1u], (it >> 1) & 1u);
            for (uint32_t t = 0; ok && t < tiles; ++t) {
                ok = wait(&bars->q_full[t], n_q[t]++ & 1u);
                if (!ok) break;
                fence_after();
                qk(t, it & 1u);
            }
            if (!ok) break;
            tc_commit(&bars->k_empty[it & 1u]);
            for (uint32_t j = 0; ok && j < seg.take; ++j, ++it) {
                const uint32_t st = it & 1u, sn = (it + 1) & 1u;
                for (uint32_t t = 0; t < tiles; ++t) {
                    ok = wait(&bars->p_full[t], n_p[t]++ & 1u) && (t != 0 || wait(&bars->v_full[st], (it >> 1) & 1u));
                    if (!ok) break;
                    fence_after();
                    const uint32_t vb = base + G::kOffV + st * G::kK;
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        tc_mma_ts(tmem + 256u + t * 128u, tmem + t * 128u + kk * 8u,
                                  desc_sw128(vb + (kk >> 2) * (D * 128u) + (kk & 3) * 32u), G::kIdescPV, (j | kk) != 0);
                    tc_commit(&bars->o_done[t]);
                    if (t == tiles - 1) tc_commit(&bars->v_empty[st]);
                    if (j + 1 < seg.take) {
                        if (t == 0) {
                            ok = wait(&bars->k_full[sn], ((it + 1) >> 1) & 1u);
                            if (!ok) break;
                            fence_after();
                        }
                        qk(t, sn);
                        if (t == tiles - 1) tc_commit(&bars->k_empty[sn]);
                    }
                }
            }
        }
        if (!ok) {
            // unwinding: the products in flight end before their memory is given back
            tc_commit(&bars->drained);
            const uint64_t t0 = clock64();
            while (!pipe::mbar_try(&bars->drained, 0) && clock64() - t0 < pipe::kWaitCycles) {}
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kWarpsT - 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

template <int D, typename QT> __global__ void __launch_bounds__(128) attn_tc_join_kernel(const __grid_constant__ AttnArgs a)
{
    wait_previous();
    for (uint32_t rr = threadIdx.x >> 5; rr < 32; rr += 4) join_row<kTcRows, D, QT>(a, a.desc, a.part, blockIdx.x, blockIdx.y * 32 + rr);
}

template <int D, int FMT, typename QT> cudaError_t launch_tc_one(const AttnArgs &a, uint32_t grid, cudaStream_t s)
{
    auto kernel = attn_tc_kernel<D, FMT, QT>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(kernel, TcGeo<D>::kSmem, ready);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kThreadsT, TcGeo<D>::kSmem, s>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_behind(attn_tc_join_kernel<D, QT>, dim3(grid, kTcRows / 32), dim3(128), 0, s, a);
}

template <int D> cudaError_t launch_tc_dim(const AttnArgs &a, uint32_t fmt, int elem, uint32_t grid, cudaStream_t s)
{
    if (elem == HXQ_ELEM_BF16)
        return fmt == HXQ_KV_INT8 ? launch_tc_one<D, HXQ_KV_INT8, __nv_bfloat16>(a, grid, s)
                                  : launch_tc_one<D, HXQ_KV_E4M3, __nv_bfloat16>(a, grid, s);
    return fmt == HXQ_KV_INT8 ? launch_tc_one<D, HXQ_KV_INT8, __half>(a, grid, s) : launch_tc_one<D, HXQ_KV_E4M3, __half>(a, grid, s);
}

cudaError_t launch_attn_tc(const AttnArgs &a, uint32_t D, uint32_t fmt, int elem, uint32_t grid, cudaStream_t s)
{
    return D == 64 ? launch_tc_dim<64>(a, fmt, elem, grid, s) : launch_tc_dim<128>(a, fmt, elem, grid, s);
}

}  // namespace serving
}  // namespace hxq
