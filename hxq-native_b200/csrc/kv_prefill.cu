// kv_prefill.cu -- attention over the 8-bit cache for many query rows per
// key (prompts, chunks of prompts) on tcgen05.
//
// The mathematics is kv_attention.cu's: products on codes alone, block scales
// inside the exponent and the row sums.  A CTA takes 256 rows (tokens x heads
// of a group) of one (request, cache head), two tiles of 128, against 128 keys
// at a time:
//   warps 0-15  two threads a row (tile = warp / 8), each for half of the keys:
//               Q scaled into f16 and into shared memory once, then for every
//               128 keys the scores out of tensor memory, exp2, weights back
//               into tensor memory as f16 over the scores' columns; at the
//               end the row out, through Q's place so that stores coalesce;
//   warps 16-19 codes: shared memory (as they are in the cache) -> f16 ->
//               shared memory, keys [key][dim] and values transposed
//               [dim][key], both K-major with 128-byte swizzle;
//   warp 20     one thread issues S = Q K^T (both operands in shared memory)
//               and O += P V (P in tensor memory);
//   warps 21,23 a lane for every 16 keys looks up their block, copies its
//               codes to shared memory (cp.async.bulk) and its scales, one
//               warp for keys and one for values;
//   warp 22     one thread cuts the CTA's range into segments for the others.
// The two tiles take turns: while one is at its exponentials, the tensor
// cores work for the other.  Tensor memory, all 512 columns, one CTA an SM:
// heads of 128 have a buffer of 128 scores for each tile and two accumulators,
// heads of 64 a third buffer, so that the next scores of a tile are computed
// while it is at these (chunks below 115 -> 107 us).
//
// The running maximum is lazy: it is raised, and O rescaled, only where a
// weight would grow by more than 2^8, which after the first keys is rare,
// so that the rescale needs no warps of its own.
//
// Bound by what passes between the warps in a step: scores to the rows' threads,
// weights back, the next scores behind the weights' product (about 4,900 cycles
// a step of two tiles, where the tensor pipe needs 2,060, the exponentials
// 2,050 and the conversion's shared memory traffic about 2,500).  Three prompts
// of up to 4096 rows, 32 heads of 128, int8: 375 to 382 us a call, 640 TFLOP/s (37%
// of the measured matrix rate; tensor pipe active 33% of the time, instructions
// issued in 61% of the cycles); two chunks of 512 rows x 40 heads of 64 over a
// window of 4096 keys, e4m3: 109 us.  A second issuing warp, one a
// tile, cost (462 -> 490 us at the time).
//
// Work is cut and joined as in kv_attention.cu, with granules of 128 keys.
// Every wait is bounded by the clock; one that runs out is recorded and the CTA
// unwinds.
#include "kv_attention.cuh"

#include "tc_pipe.cuh"

namespace hxq {
namespace serving {

constexpr int kKeys = 128;                 // keys of a step
constexpr int kTile = 128;                 // rows of a tile
constexpr int kFixedT = 3;                 // steps that a unit costs by itself (the prompts above and the chunks: 2: 395, 108.4 us, 3: 375, 108.8, 4: 380, 108.9)
constexpr int kSoftWarps = 16, kConvWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kConvWarps, kLoadWarp = kMmaWarp + 1, kPlanWarp = kMmaWarp + 2;
constexpr int kWarpsT = kMmaWarp + 4;       // six warpgroups
// Registers: launched with 80 a thread, 61,440 in all; the rows' threads hold
// 16 scores and the next 16. 512 x 88 + 128 x 64 + 128 x 64 = 61,440.
constexpr int kRegsSoft = 88, kRegsConv = 64, kRegsRest = 64;
constexpr int kThreadsT = kWarpsT * 32;
constexpr int kSegSlots = 2;
constexpr float kRaise = 8.0f;             // log2 of the largest weight (less the lift) before the maximum is raised

template <int D> struct TcGeo {
    static constexpr int kQ = kTile * D * 2;           // bytes of a tile of Q
    static constexpr int kK = kKeys * D * 2;           // of a step's keys, and of its values
    static constexpr int kRaw = kKeys * D;             // bytes of their codes
    static constexpr int kOffK = 2 * kQ, kOffV = kOffK + 2 * kK, kOffRaw = kOffV + 2 * kK, kOffS = kOffRaw + 2 * kRaw;
    // Buffers of scores: one a tile, and one more where heads of 64 leave the
    // columns for it: then the scores of a tile's next step are there when it
    // is done with this one's. Their steps' scales are kept that much longer.
    static constexpr int kBufs = D == 64 ? 3 : 2, kScaleSlots = D == 64 ? 8 : 4, kColO = 128 * kBufs;
    static constexpr int kOffSeg = kOffS + kScaleSlots * 8 * 16, kOffBar = kOffSeg + kSegSlots * 64;
    // A float for every row of both tiles and halves, in which the two warps of a row exchange their maxima. Two of them,
    // taken in turn, where a tile's next scores may be there before both warps are done with this step's: a warp then
    // writes the next step's while its partner reads this one's, and the barrier of that next step is what lies between
    // this read and the write after it. With a buffer a tile the next scores follow all eight warps' weights.
    static constexpr int kTops = kBufs == 2 ? 1 : 2, kTop = 2 * 2 * kTile;
    static constexpr int kOffTop = kOffBar + 320;
    static constexpr int kSmem = kOffTop + kTops * kTop * 4;
    static_assert(kSmem <= 232448, "shared memory");
    static_assert(kOffS - 1024 >= 4 * (HXQ_ATTENTION_MAX_REQUESTS + 1) && sizeof(RangeShared<kWarpsT>) <= 1024, "room for the scan");
    static constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
    static constexpr uint32_t kIdescPV = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
};

// K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// The products' warp runs as one, so that descriptors stay in uniform
// registers; `one` is true in the lane that issues.
__device__ __forceinline__ void tc_mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
                 : "memory");
}

__device__ __forceinline__ void tc_mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
                 : "memory");
}

__device__ __forceinline__ void tc_commit(uint32_t one, uint64_t *bar)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(pipe::smem_u32(bar)), "r"(one)
                 : "memory");
}

__device__ __forceinline__ uint32_t elect_one()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
    return r;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tm_st8(uint32_t taddr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

__device__ __forceinline__ void tm_ld16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct Bars {
    uint64_t q_full[2], s_full[2][3], p_full[3], o_done[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t rawk_full, rawk_empty, rawv_full, rawv_empty, seg_full[kSegSlots], seg_empty[kSegSlots], drained;
    uint32_t tmem, gave_up;
    // of a raw step (by its parity): keys up to the range's last (0: no more steps) and, in the upper half, those in front
    // of its first; value groups that count as 0
    uint32_t live[2], zero[2][8];
};
static_assert(sizeof(Bars) <= 320, "room for the barriers");

// What the warps need of a segment; take 0: no more of them.
struct SegInfo {
    uint32_t take, take0;            // steps, and those that tile 0 takes part in
    uint32_t key0, hi, r0, r1, q0, h, b;
    int32_t before;                  // position of the request's first row
    uint32_t len;
    uint16_t whole, front;           // front: keys of the first step that no row sees, a window being behind them
    int4 cut;                        // for the joining kernel, where the segment begins a unit and doesn't end it
};
static_assert(sizeof(SegInfo) == 64, "a slot");

__device__ __forceinline__ void named_sync(uint32_t id, uint32_t threads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The same, and whether `ok` holds in every one of the threads.
__device__ __forceinline__ bool named_all(uint32_t id, uint32_t threads, bool ok)
{
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all)
                 : "r"(id), "r"(threads), "r"((uint32_t)ok)
                 : "memory");
    return all != 0;
}

// Largest of 16 scores.
__device__ __forceinline__ float largest16(const uint32_t *s)
{
    float m[5];
#pragma unroll
    for (int i = 0; i < 5; ++i)
        m[i] = fmaxf(fmaxf(__uint_as_float(s[3 * i]), __uint_as_float(s[3 * i + 1])), __uint_as_float(s[3 * i + 2]));
    return fmaxf(fmaxf(fmaxf(m[0], m[1]), m[2]), fmaxf(fmaxf(m[3], m[4]), __uint_as_float(s[15])));
}

// Weights of 16 scores, as f16 pairs (MASK: 0 for keys that the row may not
// see, whatever the scales of their block); their sum is returned.
template <bool MASK>
__device__ __forceinline__ float weigh16(const uint32_t *s, float f, float off, uint32_t *p, int32_t key, int32_t pos, int32_t floor)
{
    const uint64_t f2 = pack2(f, f), off2 = pack2(off, off);
    uint64_t sum2 = 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        float2 t = unpack2(fma2(pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), f2, off2));
        if (MASK) {
            if (key + i > pos || key + i <= floor) t.x = -INFINITY;
            if (key + i + 1 > pos || key + i + 1 <= floor) t.y = -INFINITY;
        }
        const float w0 = ex2(t.x), w1 = ex2(t.y);
        sum2 = i == 0 ? pack2(w0, w1) : add2(sum2, pack2(w0, w1));
        const __half2 h = __floats2half2_rn(w0, w1);
        p[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
    }
    const float2 sum = unpack2(sum2);
    return sum.x + sum.y;
}

// The largest s + log2 vs of a row's 64 scores (of those it may see).  Scales
// are not negative; NaN is passed over here.
template <bool MASK>
__device__ __forceinline__ float largest64(uint32_t tS, const float4 *sc, float fac, uint32_t key0, int32_t pos, int32_t floor)
{
    float top = -INFINITY;
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        uint32_t s[16];
        tm_ld16(tS + g * 16, s);
        wait_ld();
        if (MASK) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int32_t key = (int32_t)key0 + g * 16 + i;
                if (key > pos || key <= floor) s[i] = 0xff800000u;   // -infinity
            }
        }
        top = fmaxf(top, fmaf(largest16(s), fac * sc[g].x, sc[g].y));
    }
    return top;
}

// Their weights as f16 over the first half of their columns (16 scores are
// read, then 8 columns written); returns the sum of weight / vs.
template <bool MASK>
__device__ __forceinline__ float weigh64(uint32_t tS, const float4 *sc, float fac, float ms, uint32_t key0, int32_t pos, int32_t floor)
{
    float l = 0.0f;
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        uint32_t s[16], p[8];
        tm_ld16(tS + g * 16, s);
        wait_ld();
        const float sum = weigh16<MASK>(s, fac * sc[g].x, sc[g].y - ms, p, (int32_t)key0 + g * 16, pos, floor);
        // a row that sees none of the 16 keys takes nothing from their block, whatever its scale
        l += MASK && sum == 0.0f ? 0.0f : sum * sc[g].z;
        tm_st8(tS + g * 8, p);
    }
    return l;
}

template <int D, int FMT, typename QT>
__global__ void __launch_bounds__(kThreadsT, 1) attn_tc_kernel(const __grid_constant__ AttnArgs a)
{
    using G = TcGeo<D>;
    extern __shared__ __align__(1024) uint8_t smem[];   // the kernel has no other shared memory: it begins on 1024
    RangeShared<kWarpsT> &sh = *reinterpret_cast<RangeShared<kWarpsT> *>(smem + G::kOffS - 1024);
    SegInfo *segs = reinterpret_cast<SegInfo *>(smem + G::kOffSeg);
    Bars *bars = reinterpret_cast<Bars *>(smem + G::kOffBar);
    float4 *scales = reinterpret_cast<float4 *>(smem + G::kOffS);   // [slot][16-key group]: ks, log2 vs, 1 / vs
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = pipe::smem_u32(smem);

    let_next_start();
    if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    Range range;
    if (!find_range<kWarpsT, kTcRows, kKeys, kFixedT>(a, sh, reinterpret_cast<uint32_t *>(smem), false, range)) {
        wait_previous();
        return;
    }
    if (tid == 0) {
        bars->gave_up = 0;
        for (int t = 0; t < 2; ++t) {
            pipe::mbar_init(&bars->q_full[t], kSoftWarps / 2);   // one arrival a warp
            pipe::mbar_init(&bars->o_done[t], 1);
            pipe::mbar_init(&bars->k_full[t], kConvWarps);
            pipe::mbar_init(&bars->k_empty[t], 1);
            pipe::mbar_init(&bars->v_full[t], kConvWarps);
            pipe::mbar_init(&bars->v_empty[t], 1);
        }
        for (int b = 0; b < 3; ++b) {
            for (int t = 0; t < 2; ++t) pipe::mbar_init(&bars->s_full[t][b], 1);
            pipe::mbar_init(&bars->p_full[b], kSoftWarps / 2);
        }
        pipe::mbar_init(&bars->rawk_full, 8);
        pipe::mbar_init(&bars->rawk_empty, kConvWarps);
        pipe::mbar_init(&bars->rawv_full, 8);
        pipe::mbar_init(&bars->rawv_empty, kConvWarps);
        for (int i = 0; i < kSegSlots; ++i) {
            pipe::mbar_init(&bars->seg_full[i], 1);
            pipe::mbar_init(&bars->seg_empty[i], kSoftWarps + 3);   // the rows' warps, both loads, products
        }
        pipe::mbar_init(&bars->drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pipe::smem_u32(&bars->tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bars->tmem;

    // Where a wait runs out, the CTA unwinds: the other waits follow (gave_up), a warp takes a wait's outcome as one, and the
    // warps of the rows meet at every barrier of theirs first, so that they leave the loops together.
    auto wait = [&](uint64_t *bar, uint32_t parity) { return bounded_wait(bar, parity, &bars->gave_up, a); };
    bool ok = true;
    if (warp < kSoftWarps) {
        // ------------------------------------------------------- rows
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
        const uint32_t t = warp >> 3, hf = warp >> 2 & 1u, rr = tid & (kTile - 1);   // tile, half of the keys, row of the tile
        const uint32_t lanes = (warp & 3u) << 21;                      // this warp's 32 lanes of tensor memory
        const uint32_t tS0 = tmem + lanes + hf * 64u;
        const uint32_t tO = tmem + lanes + G::kColO + t * D + hf * (D / 2);
        const uint32_t pair = 1 + t * 4 + (warp & 3u), whole_tile = 9 + t;           // named barriers: 64 and 256 threads
        float *tops = reinterpret_cast<float *>(smem + G::kOffTop) + t * 2 * kTile;
        const uint32_t qt = base + t * G::kQ;
        uint32_t n_s = 0;                                              // steps of this tile so far
        uint32_t turns = 0;                                            // of each buffer's barrier, as a parity
        uint32_t step0 = 0, use0 = 0;                                  // CTA's steps, and tiles' steps, before this segment
        for (uint32_t si = 0;; ++si) {
            const SegInfo &seg = segs[si % kSegSlots];
            ok = named_all(whole_tile, 2 * kTile, wait(&bars->seg_full[si % kSegSlots], si / kSegSlots & 1u));
            if (!ok || seg.take == 0) break;
            const uint32_t take = t == 0 ? seg.take0 : seg.take, key_first = seg.key0;
            const uint32_t tr0 = seg.r0 + t * kTile, r1 = seg.r1;
            const bool two = r1 - seg.r0 > (uint32_t)kTile;
            const uint32_t both = two ? seg.take0 : 0;                 // steps that both tiles take part in
            if (tr0 >= r1) {
                step0 += seg.take;
                use0 += seg.take;
                __syncwarp();
                if (lane == 0) pipe::mbar_arrive(&bars->seg_empty[si % kSegSlots]);
                continue;
            }
            const uint32_t tr1 = min(tr0 + kTile, r1);
            const int32_t before = seg.before, last = (int32_t)seg.len - 1;
            auto position = [&](uint32_t rw) { return a.causal ? before + (int32_t)token_of(a, rw) : last; };
            auto key_floor = [&](int32_t at) { return a.window ? (int32_t)max((int64_t)at - (int64_t)a.window, (int64_t)-1) : -1; };
            const int32_t pos_first = position(tr0), pos_last = position(tr1 - 1), pos = tr0 + rr < tr1 ? position(tr0 + rr) : pos_last;
            const int32_t floor_last = key_floor(pos_last), floor = key_floor(pos);
            // Q: a row's largest into [2^14, 2^15), 0 and non-finite rows as they are. D / 8 lanes a row.
            {
                constexpr uint32_t kLanes = D / 8, kRowsQ = 32 / kLanes;
                const uint32_t c = lane % kLanes;
                // rows as they are into their places, all under way at once; then each lane turns its own pieces.
                // (Rolled loops: this runs once a segment, and straight code of its length misses the instruction
                // cache all the way: 11,500 cycles a segment where this takes a third.)
                auto place = [&](uint32_t r) { return qt + (c >> 3) * (kTile * 128u) + r * 128u + (((c & 7u) ^ (r & 7u)) << 4); };
#pragma unroll 1
                for (uint32_t i = 0; i < 16; i += kRowsQ) {
                    const uint32_t r = (warp & 7u) * 16 + i + lane / kLanes, row = min(tr0 + r, tr1 - 1), tk = token_of(a, row);
                    const QT *src = static_cast<const QT *>(a.q) + (int64_t)(seg.q0 + tk) * a.q_st + (int64_t)(seg.h * a.G + (row - tk * a.G)) * a.q_sh + c * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place(r)), "l"(src), "r"(tr0 + r < tr1 ? 16 : 0) : "memory");
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
#pragma unroll 1
                for (uint32_t i = 0; i < 16; i += kRowsQ) {
                    const uint32_t r = (warp & 7u) * 16 + i + lane / kLanes;
                    const uint4 v = pipe::lds128(place(r));
                    const QT *e = reinterpret_cast<const QT *>(&v);
                    uint32_t top = 0;
#pragma unroll
                    for (int u = 0; u < 8; ++u) top = max(top, __float_as_uint(fabsf(Elem<QT>::to(e[u]))));
#pragma unroll
                    for (uint32_t d = 1; d < kLanes; d <<= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
                    const int32_t e2 = (int32_t)(top >> 23) - 127;
                    const int32_t shift = (top == 0 || e2 == 128) ? 0 : max(-113, min(126, 14 - e2));
                    const float m = __uint_as_float((uint32_t)(127 + shift) << 23);
                    uint32_t w[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const __half2 h = __floats2half2_rn(Elem<QT>::to(e[2 * u]) * m, Elem<QT>::to(e[2 * u + 1]) * m);
                        w[u] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    sts128(place(r), w[0], w[1], w[2], w[3]);
                    if (c == 0) tops[r] = a.scale_log2 * __uint_as_float((uint32_t)(127 - shift) << 23);
                }
                pipe::async_proxy_fence();
                __syncwarp();
                if (lane == 0) pipe::mbar_arrive(&bars->q_full[t]);
            }
            named_sync(whole_tile, 2 * kTile);
            const float fac = tops[rr];
            named_sync(whole_tile, 2 * kTile);
            float M = -INFINITY, l = 0.0f;
            for (uint32_t j = 0; j < take; ++j) {
                const uint32_t key0 = key_first + j * kKeys + hf * 64u;
                // The buffer: the tile's own, or all in the order of the products. Its barrier is one of this tile alone:
                // a tile that a segment does not have is several turns of the buffers ahead, of its own barriers none.
                const uint32_t use = use0 + (j < both ? 2 * j + t : both + j);
                const uint32_t buf = G::kBufs == 2 ? t : use % 3u, tS = tS0 + buf * 128u;
                ok = ok && __all_sync(~0u, wait(&bars->s_full[t][buf], turns >> buf & 1u));
                turns ^= 1u << buf;
                fence_after();
                const float4 *sc = scales + ((step0 + j) & (G::kScaleSlots - 1)) * 8 + hf * 4;
                const bool all = (int32_t)(key0 + 63) <= pos_first && (int32_t)key0 > floor_last;
                // and of the other half's; NaN, which no maximum is, from a warp whose wait ran out
                float top = __uint_as_float(0x7fffffffu);
                if (ok) top = all ? largest64<false>(tS, sc, fac, key0, pos, floor) : largest64<true>(tS, sc, fac, key0, pos, floor);
                float *now = tops + (j & (G::kTops - 1)) * G::kTop;
                now[hf * kTile + rr] = top;
                named_sync(pair, 64);
                const float others = now[(hf ^ 1u) * kTile + rr];
                ok = ok && others == others;
                if (!ok) break;
                top = fmaxf(top, others);
                if (__any_sync(~0u, top > M + kRaise)) {
                    // raise the maximum (all rows of the warp; the other half's warp does the same), O and l with it
                    const float to = fmaxf(M, top), al = to == -INFINITY ? 1.0f : ex2(M - to);
                    M = to;
                    l *= al;
                    if (j > 0) {
                        ok = __all_sync(~0u, wait(&bars->o_done[t], (n_s - 1) & 1u));
                        if (!ok) continue;   // the partner learns of it in the next step, or behind the last
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[16];
                            tm_ld16(tO + c * 16, o);
                            wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                            tm_st16(tO + c * 16, o);
                        }
                        wait_st();
                    }
                }
                const float ms = (M == -INFINITY ? 0.0f : M) - kLift;
                l += all ? weigh64<false>(tS, sc, fac, ms, key0, pos, floor) : weigh64<true>(tS, sc, fac, ms, key0, pos, floor);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) pipe::mbar_arrive(&bars->p_full[buf]);
                ++n_s;
            }
            step0 += seg.take;
            use0 += both + seg.take;
            ok = named_all(whole_tile, 2 * kTile, ok && wait(&bars->o_done[t], (n_s - 1) & 1u));
            if (!ok) break;
            fence_after();
            // the products are done: Q's place takes the halves' sums, then the rows on their way out
            float *sums = reinterpret_cast<float *>(smem + t * G::kQ);
            sums[hf * kTile + rr] = l;
            named_sync(whole_tile, 2 * kTile);
            l = sums[rr] + sums[kTile + rr];
            named_sync(whole_tile, 2 * kTile);
            const uint32_t whole = seg.whole, q0 = seg.q0, head0 = seg.h * a.G;
            // rows of this warp, 16-byte columns: [half of a row's 16][row][8, swizzled] for heads of 128, [row][8] for 64
            auto place = [&](uint32_t r, uint32_t c) {   // c: column within this half's
                return D == 128 ? qt + hf * (kTile * 128u) + r * 128u + ((c ^ (r & 7u)) << 4)
                                : qt + r * 128u + (((hf * 4 + c) ^ (r & 7u)) << 4);
            };
            constexpr uint32_t kCols = D / 16, kRowsO = 32 / kCols;    // 16-byte columns of a half row; rows a warp moves at a time
            const uint32_t rw = (warp & 3u) * 32, lr = lane / kCols, lc = lane % kCols;
            if (whole) {
                const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
                for (uint32_t c = 0; c < D / 32; ++c) {
                    uint32_t o[16], w[8];
                    tm_ld16(tO + c * 16, o);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        QT e[2] = {Elem<QT>::from(__uint_as_float(o[2 * i]) * f), Elem<QT>::from(__uint_as_float(o[2 * i + 1]) * f)};
                        w[i] = *reinterpret_cast<const uint32_t *>(e);
                    }
                    sts128(place(rr, 2 * c), w[0], w[1], w[2], w[3]);
                    sts128(place(rr, 2 * c + 1), w[4], w[5], w[6], w[7]);
                }
                __syncwarp();
#pragma unroll 1
                for (uint32_t i = 0; i < 32; i += kRowsO) {
                    const uint32_t r = rw + i + lr, row = tr0 + r;
                    if (row < tr1) {
                        const uint32_t tk = token_of(a, row);
                        const uint4 v = pipe::lds128(place(r, lc));
                        QT *dst = static_cast<QT *>(a.out) + (int64_t)(q0 + tk) * a.o_st + (int64_t)(head0 + row - tk * a.G) * a.o_sh +
                                  hf * (D / 2) + lc * 8;
                        if ((((uintptr_t)dst) & 15u) == 0) *reinterpret_cast<uint4 *>(dst) = v;
                        else {
#pragma unroll
                            for (int u = 0; u < 8; ++u) dst[u] = reinterpret_cast<const QT *>(&v)[u];
                        }
                    }
                }
                if (hf == 0 && a.lse && tr0 + rr < tr1) {
                    const uint32_t tk = token_of(a, tr0 + rr);
                    a.lse[(size_t)(q0 + tk) * a.Hq + head0 + (tr0 + rr - tk * a.G)] =
                        l == 0.0f ? -INFINITY : (M - kLift + log2f(l)) * 0.69314718055994531f;
                }
            } else {
                float *part = a.part + (size_t)(2 * blockIdx.x + (seg.cut.x ? 1 : 0)) * part_floats<kTcRows, D>();
#pragma unroll 1
                for (uint32_t k = 0; k < 2; ++k) {   // a quarter of the row's columns at a time
#pragma unroll 1
                    for (uint32_t c = 0; c < D / 64; ++c) {
                        uint32_t o[16];
                        tm_ld16(tO + k * (D / 4) + c * 16, o);
                        wait_ld();
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) sts128(place(rr, 4 * c + i), o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (uint32_t i = 0; i < 32; i += kRowsO) {
                        const uint32_t r = rw + i + lr;
                        if (tr0 + r < tr1)
                            *reinterpret_cast<uint4 *>(part + (size_t)(t * kTile + r) * D + hf * (D / 2) + k * (D / 4) + lc * 4) =
                                pipe::lds128(place(r, lc));
                    }
                    __syncwarp();
                }
                if (hf == 0 && tr0 + rr < tr1) {
                    part[kTcRows * D + t * kTile + rr] = M;
                    part[kTcRows * D + kTcRows + t * kTile + rr] = l;
                }
                if (seg.cut.x && tid == 0) a.desc[blockIdx.x] = seg.cut;
            }
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bars->seg_empty[si % kSegSlots]);
            fence_before();   // O is read before the next segment's products, which wait for its weights
            named_sync(whole_tile, 2 * kTile);   // every row is on its way out: Q's place is free
        }
    } else if (warp < kSoftWarps + kConvWarps) {
        // ------------------------------------------------------- codes
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConv));
        const uint32_t cw = warp - kSoftWarps;
        // Keys: a lane takes 8 codes, one 16-byte column; the lanes of a row
        // side by side, 1024 / D rows at a time, so row & 7 stays
        constexpr uint32_t kLanesK = D / 8, kRowsK = 32 / kLanesK;
        const uint32_t kc = lane % kLanesK, kr = cw * kRowsK + lane / kLanesK;
        const uint32_t k_src = base + G::kOffRaw + kr * D + kc * 8;
        const uint32_t k_dst = (kc >> 3) * (kKeys * 128u) + kr * 128u + (((kc & 7u) ^ (kr & 7u)) << 4);
        constexpr int kNK = kKeys / (4 * kRowsK);              // 16 or 8 loads a step
        // Values: a lane takes 4 dims of 8 keys. Position i of a word holds dim
        // vd + (i + turn) % 4, so that the 8 lanes of a store phase write 8
        // different 16-byte columns; in heads of 64 the upper lanes take
        // their keys in the order 1, 0, 3, 2, .. to read the other banks
        constexpr uint32_t kLanesV = D / 4;
        constexpr int kNV = 16 * kLanesV / 128;                // 4 or 2 groups of 8 keys a step
        const uint32_t vd = (lane % kLanesV) * 4, vg = cw * (32 / kLanesV) + lane / kLanesV, swap = lane / kLanesV;
        const uint32_t turn = (lane >> 1) & 3u;
        uint32_t sel[2], v_dst[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t k = (turn + i) & 3u, dim = vd + k;
            const uint32_t pair = swap ? (k + 4) | k << 4 : k | (k + 4) << 4;   // bytes k of the two keys
            sel[i >> 1] = (i & 1) ? sel[i >> 1] | pair << 8 : pair;
            v_dst[i] = dim * 128u + ((vg & 7u) ^ (dim & 7u)) * 16u;
        }
        constexpr uint32_t kStepV = 16 / kNV;                  // groups between a lane's
        const uint32_t v_src = base + G::kOffRaw + G::kRaw + vg * 8 * D + vd;
        for (uint32_t it = 0;; ++it) {
            const uint32_t st = it & 1u, par = (it >> 1) & 1u;
            ok = __all_sync(~0u, wait(&bars->rawk_full, it & 1u));
            if (!ok) break;
            const uint32_t range = bars->live[st], live = range & 0xffffu, front = range >> 16;
            if (live == 0) break;
            if (it >= 2) ok = __all_sync(~0u, wait(&bars->k_empty[st], par ^ 1u));
            if (!ok) break;
            const uint32_t kb = base + G::kOffK + st * G::kK + k_dst;
#pragma unroll 4
            for (int i = 0; i < kNK; ++i) {
                uint2 w = pipe::lds64(k_src + i * (4 * kRowsK * D));
                const uint32_t r16 = (kr + i * 4 * kRowsK) & ~15u;
                if (range != kKeys && (r16 >= live || r16 + 16 <= front)) w = make_uint2(0, 0);   // not copied
                uint32_t h[4];
                codes_to_f16<FMT>(w.x, h[0], h[1]);
                codes_to_f16<FMT>(w.y, h[2], h[3]);
                sts128(kb + i * (4 * kRowsK * 128u), h[0], h[1], h[2], h[3]);
            }
            pipe::async_proxy_fence();
            __syncwarp();
            if (lane == 0) {
                pipe::mbar_arrive(&bars->k_full[st]);
                pipe::mbar_arrive(&bars->rawk_empty);
            }
            ok = __all_sync(~0u, wait(&bars->rawv_full, it & 1u));
            if (!ok) break;
            if (it >= 2) ok = __all_sync(~0u, wait(&bars->v_empty[st], par ^ 1u));
            if (!ok) break;
            const uint32_t vb = base + G::kOffV + st * G::kK;
#pragma unroll 1
            for (int i = 0; i < kNV; ++i) {
                const uint32_t grp = i * kStepV + vg;
                uint32_t w[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) w[u] = pipe::lds32(v_src + i * (kStepV * 8 * D) + (D == 64 ? u ^ swap : u) * D);
                const bool drop = bars->zero[st][grp >> 1] != 0;
                if (drop || grp * 8 + 8 > live || grp * 8 < front) {
                    // blocks that count as 0, and slots behind the last key or in front of the first, which may hold anything
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (drop || grp * 8 + (D == 64 ? u ^ swap : u) - front >= live - front) w[u] = 0;
                }
                uint32_t o[4][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    codes_to_f16<FMT>(__byte_perm(w[2 * u], w[2 * u + 1], sel[0]), o[0][u], o[1][u]);
                    codes_to_f16<FMT>(__byte_perm(w[2 * u], w[2 * u + 1], sel[1]), o[2][u], o[3][u]);
                }
                // groups i * kStepV + vg: the next half of the keys, and the other four columns of a half
                const uint32_t dst = vb + ((i * kStepV) >> 3) * (D * 128u), flip = ((i * kStepV) & 7u) << 4;
#pragma unroll
                for (int u = 0; u < 4; ++u) sts128(dst + (v_dst[u] ^ flip), o[u][0], o[u][1], o[u][2], o[u][3]);
            }
            pipe::async_proxy_fence();
            __syncwarp();
            if (lane == 0) {
                pipe::mbar_arrive(&bars->v_full[st]);
                pipe::mbar_arrive(&bars->rawv_empty);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        if ((warp == kLoadWarp || warp == kLoadWarp + 2) && lane < 8) {
            // --------------------------------------------------- loads: a warp for the keys, one for the values
            const bool keys = warp == kLoadWarp;
            uint64_t *raw_full = keys ? &bars->rawk_full : &bars->rawv_full, *raw_empty = keys ? &bars->rawk_empty : &bars->rawv_empty;
            const uint8_t *codes = keys ? a.k : a.v;
            uint8_t *dst = smem + G::kOffRaw + (keys ? 0 : G::kRaw) + lane * 16 * D;
            uint32_t it = 0;
            for (uint32_t si = 0; ok; ++si) {
                ok = __all_sync(0xffu, wait(&bars->seg_full[si % kSegSlots], si / kSegSlots & 1u));
                if (!ok) break;
                const SegInfo seg = segs[si % kSegSlots];
                __syncwarp(0xffu);
                if (lane == 0) pipe::mbar_arrive(&bars->seg_empty[si % kSegSlots]);
                if (seg.take == 0) break;
                const int32_t *row = a.table + (size_t)seg.b * a.width;
                // blocks are looked up two steps ahead, their scales one
                auto entry = [&](uint32_t j) -> int32_t {
                    const uint32_t key = seg.key0 + j * kKeys + lane * 16;
                    uint32_t slot;
                    return j < seg.take && key < seg.hi && (j > 0 || lane * 16 + 16 > seg.front) ? __ldg(row + block_of(a, key, slot)) : -1;
                };
                auto scales_of = [&](int32_t blk, float &ks, float &vs) {
                    ks = vs = 0.0f;
                    if ((uint32_t)blk < a.n_blocks) {
                        const size_t bh = (size_t)(uint32_t)blk * a.H + seg.h;
                        if (keys) ks = __ldg(a.ks + bh);
                        vs = __ldg(a.vs + bh);
                    }
                };
                int32_t blk = entry(0), blk1 = entry(1);
                float ks, vs;
                scales_of(blk, ks, vs);
                for (uint32_t j = 0; j < seg.take; ++j, ++it) {
                    const uint32_t key0 = seg.key0 + j * kKeys, key = key0 + lane * 16;
                    const int32_t blk2 = entry(j + 2);
                    float ks1, vs1;
                    scales_of(blk1, ks1, vs1);
                    const bool wanted = key < seg.hi && (j > 0 || lane * 16 + 16 > seg.front), in = wanted && (uint32_t)blk < a.n_blocks;
                    if (keys && wanted && !in) flag(a.status, HXQ_SERVING_BAD_BLOCK);
                    uint32_t slot;
                    block_of(a, key, slot);
                    const size_t src = (((size_t)(in ? (uint32_t)blk : 0u) * a.H + seg.h) * a.P + slot) * D;
                    float4 b = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);   // keys outside: no weight
                    bool zero = true;
                    if (in) {
                        b.x = ks;
                        value_scale(vs, b.y, b.z, zero);
                    }
                    if (it >= 1) ok = __all_sync(0xffu, wait(raw_empty, (it - 1) & 1u));
                    if (!ok) break;
                    if (keys) {
                        scales[(it & (G::kScaleSlots - 1)) * 8 + lane] = b;
                        if (lane == 0)
                            bars->live[it & 1u] = min((uint32_t)kKeys, seg.hi > key0 ? seg.hi - key0 : 1u) | (j == 0 ? (uint32_t)seg.front << 16 : 0u);
                    } else bars->zero[it & 1u][lane] = zero;
                    if (in) {
                        pipe::mbar_expect_tx(raw_full, 16 * D);
                        pipe::bulk_g2s(dst, codes + src, 16 * D, raw_full);
                    } else {
                        if (wanted) {   // in place of a block outside the cache
                            for (int i = 0; i < D; ++i) reinterpret_cast<uint4 *>(dst)[i] = make_uint4(0, 0, 0, 0);
                            pipe::async_proxy_fence();
                        }
                        pipe::mbar_arrive(raw_full);
                    }
                    blk = blk1;
                    blk1 = blk2;
                    ks = ks1;
                    vs = vs1;
                }
            }
            // the end of the work
            if (ok && it >= 1) ok = __all_sync(0xffu, wait(raw_empty, (it - 1) & 1u));
            if (keys && ok) {
                if (lane == 0) bars->live[it & 1u] = 0;
                pipe::mbar_arrive(raw_full);
            }
            if (!ok) let_copies_end();
        } else if (warp == kPlanWarp && lane == 0) {
            // --------------------------------------------------- segments
            Segment seg;
            for (uint32_t si = 0; ok; ++si) {
                const bool more = next_segment<kTcRows, kKeys, kFixedT>(a, range, seg);
                if (si >= kSegSlots) ok = wait(&bars->seg_empty[si % kSegSlots], (si / kSegSlots & 1u) ^ 1u);
                if (!ok) break;
                SegInfo &d = segs[si % kSegSlots];
                d.take = more ? seg.take : 0;
                if (more) {
                    uint32_t lo, hi0;
                    key_range(a, seg.r, seg.r0, min(seg.r0 + kTile, seg.r1), lo, hi0);
                    const uint32_t n0 = hi0 > seg.key0 ? (hi0 - seg.key0 + kKeys - 1) / kKeys : 1u;
                    d.take0 = seg.r1 - seg.r0 > (uint32_t)kTile ? min(n0, seg.take) : seg.take;
                    d.key0 = seg.key0;
                    d.hi = seg.hi;
                    d.r0 = seg.r0;
                    d.r1 = seg.r1;
                    d.q0 = seg.r.q0;
                    d.h = seg.h;
                    d.b = seg.b;
                    d.before = (int32_t)seg.r.len - (int32_t)seg.r.n;
                    d.len = seg.r.len;
                    d.whole = seg.begins && seg.take == seg.n;
                    d.front = (uint16_t)(seg.lo > seg.key0 ? seg.lo - seg.key0 : 0u);
                    d.cut = seg.begins && seg.take < seg.n ? cut_unit(range, seg) : make_int4(0, 0, 0, 0);
                }
                pipe::mbar_arrive(&bars->seg_full[si % kSegSlots]);
                if (!more) break;
            }
        } else if (warp == kMmaWarp) {
        const uint32_t one = elect_one();
        // ------------------------------------------------------- products
        uint32_t it = 0, use0 = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        // descriptors address 16-byte units
        const uint64_t q_desc = desc_sw128(base), k_desc = desc_sw128(base + G::kOffK), v_desc = desc_sw128(base + G::kOffV);
        for (uint32_t si = 0; ok; ++si) {
            ok = __all_sync(~0u, wait(&bars->seg_full[si % kSegSlots], si / kSegSlots & 1u));
            if (!ok) break;
            const uint32_t take = segs[si % kSegSlots].take, take0 = segs[si % kSegSlots].take0;
            const uint32_t tiles = segs[si % kSegSlots].r1 - segs[si % kSegSlots].r0 > (uint32_t)kTile ? 2u : 1u;
            __syncwarp();
            if (one) pipe::mbar_arrive(&bars->seg_empty[si % kSegSlots]);
            if (take == 0) break;
            // the tiles' steps in order: both tiles' while tile 0 has any, then one tile's
            const uint32_t both = tiles == 2 ? take0 : 0, uses = both + take;
            auto tile_of = [&](uint32_t u) { return u < 2 * both ? u & 1u : tiles - 1; };
            auto step_of = [&](uint32_t u) { return u < 2 * both ? u >> 1 : u - both; };
            uint32_t keys = 0, queries = 0;   // steps and tiles whose operands are there
            auto qk = [&](uint32_t t, uint32_t j, uint32_t buf) {
                const uint32_t st = (it + j) & 1u;
                if (j >= keys) {
                    ok = __all_sync(~0u, wait(&bars->k_full[st], ((it + j) >> 1) & 1u));
                    keys = j + 1;
                }
                if (ok && !(queries >> t & 1u)) {
                    ok = __all_sync(~0u, wait(&bars->q_full[t], n_q[t]++ & 1u));
                    queries |= 1u << t;
                }
                if (!ok) return;
                fence_after();
                const uint64_t qa = q_desc + t * (G::kQ >> 4), kb = k_desc + st * (G::kK >> 4);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    tc_mma_ss(one, tmem + buf * 128u, qa + ((kk >> 2) * (kTile * 8) + (kk & 3) * 2), kb + ((kk >> 2) * (kKeys * 8) + (kk & 3) * 2),
                              G::kIdescQK, kk != 0);
                tc_commit(one, &bars->s_full[t][buf]);
                if (t == 1 || j >= both) tc_commit(one, &bars->k_empty[st]);   // the step's last
            };
            for (uint32_t v = 0; ok && v < (uint32_t)G::kBufs && v < uses; ++v) {
                if (G::kBufs == 3) qk(tile_of(v), step_of(v), (use0 + v) % 3u);
                else if (v < tiles) qk(v, 0, v);
            }
            for (uint32_t u = 0; ok && u < uses; ++u) {
                const uint32_t t = tile_of(u), j = step_of(u), st = (it + j) & 1u;
                const uint32_t buf = G::kBufs == 2 ? t : (use0 + u) % 3u, turn = G::kBufs == 2 ? n_p[t]++ : (use0 + u) / 3u;
                ok = __all_sync(~0u, ((t == 1 && j < both) || wait(&bars->v_full[st], ((it + j) >> 1) & 1u)) && wait(&bars->p_full[buf], turn & 1u));
                if (!ok) break;
                fence_after();
                const uint64_t vb = v_desc + st * (G::kK >> 4);
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk)
                    tc_mma_ts(one, tmem + G::kColO + t * D, tmem + buf * 128u + (kk >> 2) * 64u + (kk & 3) * 8u, vb + ((kk >> 2) * (D * 8) + (kk & 3) * 2),
                              G::kIdescPV, (j | kk) != 0);
                tc_commit(one, &bars->o_done[t]);
                if (t == 1 || j >= both) tc_commit(one, &bars->v_empty[st]);   // the step's last
                if (G::kBufs == 3) {
                    if (u + 3 < uses) qk(tile_of(u + 3), step_of(u + 3), buf);
                } else if (j + 1 < (t == 0 ? take0 : take)) qk(t, j + 1, t);
            }
            it += take;
            use0 += uses;
        }
        if (!ok) {
            // unwinding: the products in flight end before their memory is given back
            tc_commit(one, &bars->drained);
            const uint64_t t0 = clock64();
            while (!pipe::mbar_try(&bars->drained, 0) && clock64() - t0 < pipe::kWaitCycles) {}
        }
        }
    }
    if (!ok) flag(a.status, HXQ_SERVING_TIMEOUT);
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    wait_previous();   // the kernel for few rows, beside which this one ran: the joining kernel waits for this one alone
}

template <int D, int FMT, typename QT> cudaError_t launch_tc_one(const AttnArgs &a, uint32_t grid, cudaStream_t s)
{
    auto kernel = attn_tc_kernel<D, FMT, QT>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(kernel, TcGeo<D>::kSmem, ready);
    if (e != cudaSuccess) return e;
    return launch_behind(kernel, dim3(grid), dim3(kThreadsT), TcGeo<D>::kSmem, s, a);
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
