// Causal attention of several query tokens over the 8-bit block cache, window and sinks included: flash attention on the fifth-generation tensor cores.
//
// Codes are exact as fp16; the blocks' scales stay float32 and meet the scores as a multiply-add and the softmax weights as a factor.  A key tile is 64 tokens of
// those that some query of the call sees: sinks, the window's blocks, the tail.
//
// blocks_fa_kernel: one CTA per SM takes a run of the flat sequence (lane x head group, row block, key tile): a row block each where there are few, otherwise whole row
// blocks or equal runs wherever that cuts them, by what each costs (divide()); a row block is NQ tiles of 128 rows = 128 / GP query tokens x the GP query heads of a GQA group.
//   * 8 NQ softmax warps, two rows' shares per thread: tcgen05.ld of the scores as fragments, one packed multiply-add each, ex2 (a quarter of them
//     by a polynomial), P back into tensor memory: fp16 (rounded once, a tenth of what a bfloat16 result loses to its own rounding), for fp16 tokens in two parts (one part's
//     rounding would be as large as the result's own: 0.00029 from float64 where two parts have the 0.00021 of the rounding alone; in one run of both 2048 queries over 16,384
//     tokens took 472 us with one part, 593 with two, a window of 1024 72 and 81); a row's reference maximum is looked at through its sum.  They also lay out their rows of the queries, the next row block's before they write
//     this one's results;
//   * a warp per query tile issues S = Q K^T and O += P V, scores two key tiles ahead (N = 64: 48 clocks an instruction with Q in shared memory, of 32 with it in tensor
//     memory, where there is no room for it; 620 a tile and query tile with the values' products);
//   * keys and values as fp16 operands, by one of two ways:
//     - expanded (NQ = 2; 1 at d = 256): blocks_fa_expand_kernel has written the tiles to workspace memory once, as they have to lie in shared memory, and two
//       threads keep four tiles of each in flight (bulk copies).  What many row blocks share is converted once;
//     - fused (NQ = 1): eight warps turn the codes into operands, a thread's next pieces of 16 bytes on their way in registers.  For calls of one or two row
//       tiles per lane, where writing fp16 rows and reading them back would cost more than the products.
// blocks_fa_merge_kernel joins the partials of row blocks that several CTAs worked on, in their order.
//
// Measured: 2048 queries over 16,384 tokens, 32 heads on 8, d = 128: 535 us = 960 TFLOP/s (309 at the 1668 that a large product reaches); expansion 20 and merge 19 of it.
// Bound by both together: of some 1900 clocks per pair of query tiles and key tile the tensor pipe is busy 1240 and the special-function unit 770; a score buffer is full again some
// 1600 after its weights (both query tiles' products, in one queue), and a tile's softmax takes 1350, issue slots shared with the other query tile's. Tried without gain: a warp for
// scores and another for results (574), weights in tensor-memory buffers of their own (550), the values' scale in the exponent (542), naps between looks at barriers, key tiles of 128
// tokens (663).
// Every mbarrier wait is bounded; one that runs out leaves status 114 (tq_device_status) and raises a flag that ends every other wait; copies and products in
// flight are waited for (bounded), tensor memory is freed on every path.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "blocks.cuh"
#include "fa_dev.cuh"

namespace tq {

int* decode_status_ptr();

namespace bfa {

using namespace fa;

constexpr int ERR_WAIT = 114;
constexpr int NSC = 8;                                 // tiles' scales in flight
constexpr int MAX_CTAS = 160;                          // CTAs of a launch (one per SM)
constexpr int TN = 64;                                 // tokens per key tile
// Weights reach the products as fp16, up to 2^16: a row's weights may pass its reference by 2^SLACK, the value scales are brought to [2^VS_LOG2, twice that) and may grow
// to VS_CAP.  Each row that asks for a new reference costs its query tile some 2000 clocks (2048 queries x 16,384 at SLACK 6: 570 us; 9: 554; 11: 546); what it costs at the
// other end is that a weight below 2^-18 of the reference is rounded by up to 2^-29 of it, 2^-14 in all if 32,768 tokens' weights were all such and all off one way.
constexpr int SLACK = 10, VS_LOG2 = 4;
constexpr float VS_CAP = 63.f;
constexpr int TILE_INFO = 2 * TN + 4;                  // words that go with a tile: scales, first token, end of its region

template <int D, bool FUSED> struct Plan {
    static constexpr int NQ = FUSED || D == 256 ? 1 : 2;       // query tiles per CTA
    static constexpr int SB = 2;                       // score buffers per query tile
    static constexpr int ST = D == 256 ? 2 : 4;        // key tiles (and value tiles) in shared memory
    static constexpr int NBLK = (D + 63) / 64;         // 64-column blocks of a row
    static constexpr int DP = NBLK * 64;               // columns of O (d = 96: nobody reads the last 32)
    static constexpr int SW = NQ * 8, XW = FUSED ? 8 : 2, NT = (SW + NQ + XW) * 32;    // softmax warps; MMA warps; warps that bring keys and values
    static constexpr int CH = D / 32;                  // 16-byte pieces of a tile per expanding thread (128 a side)
    static constexpr uint32_t QBLK = TM * 128u, KBLK = TN * 128u;            // bytes of a 64-column block
    static constexpr uint32_t Q_TILE = NBLK * QBLK, K_TILE = NBLK * KBLK;
    static constexpr uint32_t OFF_Q = 0, OFF_K = NQ * Q_TILE, OFF_V = OFF_K + ST * K_TILE;
    static constexpr uint32_t SC = TILE_INFO * 4, OFF_SC = OFF_V + ST * K_TILE;       // per tile float keys[TN], values[TN], int its first token, the end of its region
    static constexpr uint32_t OFF_BAR = OFF_SC + NSC * SC;
    static constexpr uint32_t OFF_SLOT = OFF_BAR + 8 * 48;                   // [0] tensor-memory base, [1] abort
    static constexpr size_t NEED = OFF_SLOT + 16 + 1024, SMEM = NEED > 116 * 1024 ? NEED : 116 * 1024;      // one CTA per SM: it takes all of the tensor memory
    static constexpr uint32_t COL_O = NQ * SB * TN;                          // scores first, then the accumulators
    static constexpr int ROWS = NQ * TM;               // of a row block
    static_assert(COL_O + NQ * DP <= 512, "tensor memory");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
enum Bars { K_FULL = 0, K_FREE = 4, V_FULL = 8, V_FREE = 12, SC_FULL = 16, SC_FREE = 24, S_FULL = 32, P_FULL = 36, O_DONE = 40, ALL_DONE = 42, Q_FULL = 44, DRAIN = 46 };       // (48 of 8 bytes)

// The key tiles of a range of query positions, in their order: sinks, the window's in blocks, the tail's
struct Tiles {
    int n_sink, low_tile, n_code, tail_tile, n;
    __host__ __device__ Tiles(const BlockAttendParams& c, int first_pos, int last_pos) {
        auto mn = [](int x, int y) { return x < y ? x : y; };
        auto mx = [](int x, int y) { return x > y ? x : y; };
        const int low = mx(0, first_pos - c.window + 1), sinks = mn(c.sinks, low), code_end = mn(last_pos + 1, c.n8);
        low_tile = mn(low, c.n8) / TN;
        const int n_win = low >= code_end ? 0 : (code_end + TN - 1) / TN - low_tile, sink_tiles = (mn(sinks, code_end) + TN - 1) / TN;
        n_sink = n_win > 0 ? mn(sink_tiles, low_tile) : sink_tiles;
        n_code = n_sink + n_win;
        tail_tile = sinks > c.n8 ? 0 : mx(low - c.n8, 0) / TN;
        n = n_code + (last_pos < c.n8 ? 0 : (last_pos + 1 - c.n8 + TN - 1) / TN - tail_tile);
    }
    __host__ __device__ bool is_tail(int t) const { return t >= n_code; }
    __host__ __device__ int tile_of(int t) const { return t < n_sink ? t : t < n_code ? low_tile + t - n_sink : tail_tile + t - n_code; }      // of the blocks, of the tail
};

struct Params {
    BlockAttendParams a;
    int lane0;                                         // first cache lane of this launch
    int HG, GP, QT, n_blk;                             // head groups, padded heads of one; query tokens per query tile; row blocks
    int ctas;
    struct Start { int job, tile; } start[MAX_CTAS + 1];       // where each CTA's run begins: (lane x head group, row block) and its key tile
    float* part;                                       // two partials per CTA: NQ * 128 rows of D + 4 floats (sums, maximum, sum of weights)
    const unsigned char* tiles;                        // expanded: per lane and key tile of the call the keys', the values'
    const float* scales;                               // ... and what goes with each
    Tiles all;                                         // the key tiles of the call
    int* status;
};

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// Sixteen codes as the two 16-byte chunks of an fp16 operand row
__device__ __forceinline__ void expand16(uint4 raw, int e4m3, uint4& lo, uint4& hi) {
    if (e4m3) {
        halves<true>(raw.x, lo.x, lo.y); halves<true>(raw.y, lo.z, lo.w); halves<true>(raw.z, hi.x, hi.y); halves<true>(raw.w, hi.z, hi.w);
    } else {
        halves<false>(raw.x, lo.x, lo.y); halves<false>(raw.y, lo.z, lo.w); halves<false>(raw.z, hi.x, hi.y); halves<false>(raw.w, hi.z, hi.w);
    }
}
// Place of 16-byte chunk `ch` (of D / 8) of row `row` in a tile of 64-column blocks, 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_place(int row, int ch) { return uint32_t(ch >> 3) * (TN * 128u) + uint32_t(row) * 128u + (uint32_t((ch ^ row) & 7) << 4); }
__device__ __forceinline__ uint32_t largest16(uint4 x) {
    const uint32_t k = 0x7fff7fffu, z = __vmaxu2(__vmaxu2(x.x & k, x.y & k), __vmaxu2(x.z & k, x.w & k));
    return max(z & 0xffffu, z >> 16);
}
__device__ __forceinline__ uint4 bf_to_half(uint4 x, float f) {
    auto two = [&](uint32_t v) { return pack_h2(__uint_as_float(v << 16) * f, __uint_as_float(v & 0xffff0000u) * f); };
    return make_uint4(two(x.x), two(x.y), two(x.z), two(x.w));
}
// A token whose values are not finite would reach rows that it is hidden from as 0 * inf: its value row is zeros, its value scale 0, its key scale (and with it the
// scores of those who see it) NaN.
__device__ __forceinline__ bool finite_scale(float v) { return fabsf(v) <= 3.4028235e38f; }

// 2^x of two values without the special-function unit, whose rate is what the softmax of a tile would otherwise wait for: 2^round(x) times a polynomial of degree 4 on
// [-1/2, 1/2] that is 1 at 0, fitted to the least relative error (2^-18.4).  x goes through [0, 1], whose steps are 2^-17 of x's range there: the whole is within 2^-16.8 of 2^x,
// a thirtieth of a weight's rounding to fp16.  x outside [-127, 127] counts as the end it passed; at -127 and below the result is below 2^-126.  NaN counts as the lower end: scores are NaN for a whole token
// or not at all (a scale that is NaN, a query that is; codes are finite), and the columns whose exponentials are ex2's tell.
__device__ __forceinline__ float unit_of(float x) {        // [-127, 127] -> [0, 1], clamped (NaN: 0)
    float y;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(x), "f"(1.f / 254.f), "f"(0.5f));
    return y;
}
__device__ __forceinline__ u64 ex2_by_fma(float x0, float x1) {
    constexpr float ROUND = 12582912.f;                    // 3 * 2^22: the integer part ends up in the low bits
    const u64 y = pk(unit_of(x0), unit_of(x1)), width = pk(254.f, 254.f);
    const u64 t = fma2(y, width, pk(ROUND - 127.f, ROUND - 127.f));
    const u64 f = fma2(y, width, fma2(t, pk(-1.f, -1.f), pk(ROUND - 127.f, ROUND - 127.f)));
    u64 p = fma2(f, pk(0.00958285294f, 0.00958285294f), pk(0.0559064262f, 0.0559064262f));
    p = fma2(p, f, pk(0.240240991f, 0.240240991f));
    p = fma2(p, f, pk(0.693124175f, 0.693124175f));
    p = fma2(p, f, pk(1.f, 1.f));
    float p0, p1, t0, t1;
    upk(p, p0, p1);
    upk(t, t0, t1);
    return pk(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23)), __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23)));
}
constexpr int POLY_EVERY = 4;                          // (none 551 us for 2048 queries x 16,384, every fourth pair 539, every second 570: issue)

template <int D, bool FUSED, bool FINE>
__global__ void __launch_bounds__(Plan<D, FUSED>::NT, 1) blocks_fa_kernel(const __grid_constant__ Params p) {
    using P = Plan<D, FUSED>;
    constexpr int NQ = P::NQ, DP = P::DP, SB = P::SB, ST = P::ST;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t raw_addr = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t sbase = (raw_addr + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (sbase - raw_addr);
    volatile uint32_t* slot = reinterpret_cast<volatile uint32_t*>(smem + P::OFF_SLOT);
    auto bar = [&](int which) -> uint32_t { return sbase + P::OFF_BAR + 8u * uint32_t(which); };
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // (uniform)
    const BlockAttendParams& c = p.a;
    const int q_pos0 = c.total - c.Tq, gp_bits = 31 - __clz(p.GP);

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(K_FULL + i), FUSED ? 128 : 1); mbar_init(bar(K_FREE + i), NQ); mbar_init(bar(V_FULL + i), FUSED ? 128 : 1); mbar_init(bar(V_FREE + i), NQ);
            mbar_init(bar(S_FULL + i), 1); mbar_init(bar(P_FULL + i), 256);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(O_DONE + i), 1); mbar_init(bar(ALL_DONE + i), 1); mbar_init(bar(Q_FULL + i), 256); mbar_init(bar(DRAIN + i), 1); }
        for (int i = 0; i < NSC; ++i) { mbar_init(bar(SC_FULL + i), FUSED ? 256 : 1); mbar_init(bar(SC_FREE + i), NQ * 256); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        slot[1] = 0u;
    }
    if (warp == P::SW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + P::OFF_SLOT), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    const uint32_t tmem = __shfl_sync(0xffffffffu, slot[0], 0);

    // This CTA's run: row blocks `job` from key tile `tile` on, up to the next CTA's start
    // (a value that a lane hands round is uniform for the compiler: loops and operands in uniform registers)
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const Params::Start from{uniform(p.start[blockIdx.x].job), uniform(p.start[blockIdx.x].tile)}, to{uniform(p.start[blockIdx.x + 1].job), uniform(p.start[blockIdx.x + 1].tile)};
    struct Segment { int lane_c, hg, tq0, t_lo, n; Tiles tiles; };
    auto segment = [&](int job) -> Segment {
        const int y = job / p.n_blk, blk = job - y * p.n_blk, tq0 = blk * NQ * p.QT;
        const Tiles t(c, q_pos0 + tq0, q_pos0 + min(tq0 + NQ * p.QT, c.Tq) - 1);
        const int lo = job == from.job ? from.tile : 0, hi = job == to.job ? to.tile : t.n;
        return Segment{y / p.HG, y - y / p.HG * p.HG, tq0, lo, hi - lo, t};
    };
    const int last_job = to.tile > 0 ? to.job : to.job - 1;

    // registers for the softmax warps from the others: 640 x 96 at launch, 512 x 112 + 128 x 32 (spilled ones cost 3%)
    if constexpr (NQ == 2) {
        static_assert(P::SW * 32 == 512 && P::NT == 640, "warpgroups");
        if (warp < P::SW) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    }
    auto wait_bar = [&](int which, int phase) -> bool {
        const uint32_t addr = bar(which);
        for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
            if (mbar_try(addr, uint32_t(phase & 1))) return true;
            if ((i & 1023u) == 1023u && slot[1]) return false;
        }
        slot[1] = 1u;
        atomicCAS(p.status, 0, ERR_WAIT);
        return false;
    };
    // copies and products end (bounded) before their memory is given up, also after a wait that ran out
    auto drain = [&](int which, int phase) {
        for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try(bar(which), uint32_t(phase & 1)); ++i) {}
    };
    // score buffer of (query tile q, key tile j of the run) and the phase of its barriers
    auto sbuf = [](int q, int j) { return q * SB + j % SB; };
    auto sph = [](int j) { return j / SB; };

    if (!FUSED && warp >= P::SW + NQ) {
        // ======================= expanded tiles: one thread the keys and scales, one the values =======================
        if (lane == 0) {
            const int side = warp - P::SW - NQ, full = side ? V_FULL : K_FULL, free_ = side ? V_FREE : K_FREE;
            const uint32_t ring = sbase + (side ? P::OFF_V : P::OFF_K);
            int j = 0, asked = 0, asked_sc = 0;
            bool ok = true;
            for (int job = from.job; job <= last_job && ok; ++job) {
                const Segment g = segment(job);
                for (int i = 0; i < g.n; ++i, ++j) {
                    // ordinal of the tile among the call's
                    const int t = g.tiles.tile_of(g.t_lo + i);
                    const int ord = g.tiles.is_tail(g.t_lo + i) ? p.all.n_code + t - p.all.tail_tile : t < p.all.n_sink ? t : p.all.n_sink + t - p.all.low_tile;
                    const int64_t at = int64_t(g.lane_c) * p.all.n + ord;
                    const int st = j % ST, s = j % NSC;
                    if (j >= ST && !(ok = wait_bar(free_ + st, j / ST - 1))) break;
                    mbar_expect_tx(bar(full + st), P::K_TILE);
                    bulk_g2s(ring + st * P::K_TILE, p.tiles + (at * 2 + side) * P::K_TILE, P::K_TILE, bar(full + st));
                    asked = j + 1;
                    if (side) continue;
                    if (j >= NSC && !(ok = wait_bar(SC_FREE + s, j / NSC - 1))) break;
                    mbar_expect_tx(bar(SC_FULL + s), P::SC);
                    bulk_g2s(sbase + P::OFF_SC + s * P::SC, p.scales + at * TILE_INFO, P::SC, bar(SC_FULL + s));
                    asked_sc = j + 1;
                }
            }
            for (int i = max(0, asked - ST); i < asked; ++i) drain(full + i % ST, i / ST);
            for (int i = max(0, asked_sc - NSC); i < asked_sc; ++i) drain(SC_FULL + i % NSC, i / NSC);
        }
        __syncwarp();
    } else if (FUSED && warp >= P::SW + NQ) {
        // ======================= codes to operands: four warps the keys, four the values =======================
        const int side = (warp - P::SW - NQ) >> 2, ct = tid - (P::SW + NQ + 4 * side) * 32;                  // 0 ... 127
        const uint32_t ring = sbase + (side ? P::OFF_V : P::OFF_K);
        const int full = side ? V_FULL : K_FULL, free_ = side ? V_FREE : K_FREE;
        int j = 0;
        bool ok = true;
        for (int job = from.job; job <= last_job && ok; ++job) {
            const Segment sg = segment(job);
            const int64_t lane_c = p.lane0 + sg.lane_c;
            const uint8_t* codes = (side ? c.vc : c.kc) + lane_c * c.cap * D;
            const float* k_scales = c.ks + lane_c * (c.cap >> c.shift);
            const float* v_scales = c.vs + lane_c * (c.cap >> c.shift);
            uint4 raw[P::CH];
            float ks = 0.f, vs = 0.f;
            auto base_of = [&](int i) { return (sg.tiles.is_tail(sg.t_lo + i) ? c.n8 : 0) + sg.tiles.tile_of(sg.t_lo + i) * TN; };
            auto fetch = [&](int base, int u) {                            // piece u of a tile
                const int x = ct + 128 * u, row = x / (D / 16);
                raw[u] = make_uint4(0u, 0u, 0u, 0u);
                if (base + row < c.n8) ld_codes(raw[u], codes + (int64_t(base + row) * D + (x - row * (D / 16)) * 16));
            };
            auto fetch_scales = [&](int base) {
                const int tok = base + ct;
                ks = vs = 0.f;
                if (ct < TN && tok < c.n8) { ks = k_scales[tok >> c.shift]; vs = v_scales[tok >> c.shift]; }
            };
            if (!sg.tiles.is_tail(sg.t_lo)) {
                const int base = base_of(0);
#pragma unroll
                for (int u = 0; u < P::CH; ++u) fetch(base, u);
                fetch_scales(base);
            }
            for (int i = 0; i < sg.n; ++i, ++j) {
                const int st = j % ST, s = j % NSC;
                if (j >= ST) ok = wait_bar(free_ + st, j / ST - 1);
                if (ok && j >= NSC) ok = wait_bar(SC_FREE + s, j / NSC - 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t tile = ring + st * P::K_TILE;
                float v = 0.f;
                if (!sg.tiles.is_tail(sg.t_lo + i)) {
                    const bool more = i + 1 < sg.n && !sg.tiles.is_tail(sg.t_lo + i + 1);
                    const int next = more ? base_of(i + 1) : 0;
                    const bool fine = finite_scale(vs);
                    v = side ? (fine ? vs : 0.f) : (fine ? ks * c.scale_log2 : __uint_as_float(0x7fffffffu));
#pragma unroll
                    for (int u = 0; u < P::CH; ++u) {
                        const int x = ct + 128 * u, row = x / (D / 16), cc = x - row * (D / 16);
                        uint4 lo, hi;
                        expand16(raw[u], c.e4m3, lo, hi);
                        // every other group of four lanes writes its second chunk first: eight lanes, eight places
                        const int swap = (cc >> 2) & 1;
                        st_shared(tile + chunk_place(row, 2 * cc + swap), swap ? hi : lo);
                        st_shared(tile + chunk_place(row, 2 * cc + 1 - swap), swap ? lo : hi);
                        if (more) fetch(next, u);
                    }
                    if (more) fetch_scales(next);
                } else {
                    // 16-bit rows, bfloat16 ones under their power of two: half a warp per token, four tokens at a time.  (A thread per token took 7 us a tile.)
                    const int base = base_of(i), half = ct >> 4, l16 = ct & 15;
                    const bool bf = c.dtype == TQ_BF16;
                    constexpr int V = D > 128 ? 2 : 1;
                    const uint16_t* const rows = static_cast<const uint16_t*>(side ? c.vt : c.kt) + lane_c * c.block * D;
                    const uint16_t* const value_rows = static_cast<const uint16_t*>(c.vt) + lane_c * c.block * D;
#pragma unroll 1
                    for (int u0 = 0; u0 < TN / 8; u0 += 4) {
                        uint4 x[4][V];
                        uint32_t mx[4], mv[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int tok = base + half + 8 * (u0 + u);
                            mx[u] = mv[u] = 0;
#pragma unroll
                            for (int w = 0; w < V; ++w) {
                                x[u][w] = make_uint4(0u, 0u, 0u, 0u);
                                if (tok < c.total && l16 + 16 * w < D / 8) {
                                    const int64_t at = int64_t(tok - c.n8) * D + (l16 + 16 * w) * 8;
                                    x[u][w] = *reinterpret_cast<const uint4*>(rows + at);
                                    if (!side) mv[u] = max(mv[u], largest16(*reinterpret_cast<const uint4*>(value_rows + at)));
                                }
                            }
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int row = half + 8 * (u0 + u);
                            const bool in = base + row < c.total;
#pragma unroll
                            for (int w = 0; w < V; ++w) mx[u] = max(mx[u], largest16(x[u][w]));
                            if (side) mv[u] = mx[u];
#pragma unroll
                            for (int off = 1; off < 16; off <<= 1) {
                                mx[u] = max(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], off));
                                mv[u] = max(mv[u], __shfl_xor_sync(0xffffffffu, mv[u], off));
                            }
                            const float f = bf ? stage_scale(mx[u] << 16) : 1.f;
                            const bool fine = mv[u] < (bf ? 0x7f80u : 0x7c00u);
#pragma unroll
                            for (int w = 0; w < V; ++w) {
                                if (l16 + 16 * w >= D / 8) continue;
                                uint4 y = bf ? bf_to_half(x[u][w], f) : x[u][w];
                                if (side && !fine) y = make_uint4(0u, 0u, 0u, 0u);
                                st_shared(tile + chunk_place(row, l16 + 16 * w), y);
                            }
                            if (l16 == 0)
                                reinterpret_cast<float*>(smem + P::OFF_SC + s * P::SC)[side * TN + row] =
                                    !in ? 0.f : side ? (fine ? 1.f / f : 0.f) : (fine ? c.scale_log2 / f : __uint_as_float(0x7fffffffu));
                        }
                    }
                }
                if (ct < TN && !sg.tiles.is_tail(sg.t_lo + i)) reinterpret_cast<float*>(smem + P::OFF_SC + s * P::SC)[side * TN + ct] = v;
                if (side && ct == 0) *reinterpret_cast<int2*>(smem + P::OFF_SC + s * P::SC + 2 * TN * 4) = make_int2(base_of(i), sg.tiles.is_tail(sg.t_lo + i) ? c.total : c.n8);
                fence_proxy_async();
                mbar_arrive(bar(full + st));
                mbar_arrive(bar(SC_FULL + s));
            }
        }
        __syncwarp();
    } else if (warp >= P::SW) {
        // ======================= MMA issue: one warp per query tile, uniform =======================
        // (With one warp for both query tiles its waits and the products' issue, one after the other, were what the softmax warps waited for: 1.3 us a key tile
        // at d = 128, of 0.7 us of products.)
        const int q = warp - P::SW;
        // up to three barriers at once, a lane each
        auto wait_all = [&](int w0, int p0, int w1, int p1, int w2, int p2) -> bool {
            const uint32_t addr = bar(lane == 0 ? w0 : lane == 1 ? w1 : w2), parity = uint32_t(lane == 0 ? p0 : lane == 1 ? p1 : p2) & 1u;
            bool done = false;
            for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
                done = done || mbar_try(addr, parity);
                if (__all_sync(0xffffffffu, done)) { __syncwarp(); return true; }
                if ((i & 1023u) == 1023u && __any_sync(0xffffffffu, slot[1] != 0u)) return false;
            }
            slot[1] = 1u;
            if (lane == 0) atomicCAS(p.status, 0, ERR_WAIT);
            return false;
        };
        auto wait_one = [&](int which, int phase) { return wait_all(which, phase, which, phase, which, phase); };
        bool ok = true, any = false;
        int j0 = 0, seg = 0;
        for (int job = from.job; job <= last_job && ok; ++job, ++seg) {
            const int n = uniform(segment(job).n);
            auto issue_qk = [&](int j) {                           // S = Q K^T of key tile j
                const uint32_t s = tmem + sbuf(q, j) * TN;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(s, desc_k(sbase + P::OFF_Q + q * P::Q_TILE, P::QBLK, ks), desc_k(sbase + P::OFF_K + (j % ST) * P::K_TILE, P::KBLK, ks),
                            idesc_of(TN, false), ks > 0 ? 1u : 0u);
                umma_commit(bar(S_FULL + sbuf(q, j)));
                umma_commit(bar(K_FREE + j % ST));
            };
            auto issue_pv = [&](int j) {                           // O += P V
                const uint32_t a = tmem + sbuf(q, j) * TN;
#pragma unroll
                for (int ks = 0; ks < TN / 16; ++ks) {
                    const uint64_t v = desc_mn(sbase + P::OFF_V + (j % ST) * P::K_TILE, P::KBLK, ks);
                    umma_ts(tmem + P::COL_O + q * DP, a + ks * 8, v, idesc_of(DP, true), (j > j0 || ks > 0) ? 1u : 0u);
                    if (FINE) umma_ts(tmem + P::COL_O + q * DP, a + TN / 2 + ks * 8, v, idesc_of(DP, true), 1u);
                }
                umma_commit(bar(O_DONE + q));
                umma_commit(bar(V_FREE + j % ST));
                if (j == j0 + n - 1) umma_commit(bar(ALL_DONE + q));       // (a barrier of its own: a parity wait on O_DONE could be two phases early or one late)
            };
            ok = wait_one(Q_FULL + q, seg);
            for (int j = j0; j < j0 + min(n, SB) && ok; ++j) {
                ok = wait_one(K_FULL + j % ST, j / ST);
                if (!ok) break;
                tc_fence_after();
                any = true;
                issue_qk(j);
            }
            for (int j = j0; j < j0 + n && ok; ++j) {
                const int jn = j + SB;                             // the key tile whose scores go where P of tile j sits now
                const bool more = jn < j0 + n;
                ok = wait_all(P_FULL + sbuf(q, j), sph(j), V_FULL + j % ST, j / ST, more ? K_FULL + jn % ST : P_FULL + sbuf(q, j), more ? jn / ST : sph(j));
                if (!ok) break;
                tc_fence_after();
                issue_pv(j);
                if (more) issue_qk(jn);                            // (the tensor core takes one thread's products in order)
            }
            j0 += n;
        }
        if (any) { umma_commit(bar(DRAIN + q)); drain(DRAIN + q, 0); }     // (nobody waits for the last products of a query tile without a row)
        __syncwarp();
    } else {
        // ======================= softmax: two rows per thread, sixteen columns of each =======================
        // Scores are read as mma.sync fragments: lane 4 g + t of a warp holds columns 8 r + 2 t, + 1 of rows g and g + 8 of its sixteen.
        const int q = warp >> 3, hh = (warp >> 2) & 1, g = lane >> 2, t2 = 2 * (lane & 3);       // query tile; half of the 32 lanes
        const uint32_t t_frag = tmem + (uint32_t((warp & 3) * 32 + 16 * hh) << 16);
        const int m0 = (warp & 3) * 32 + 16 * hh, mf = q * TM + m0 + (lane >> 2);                // the warp's first row in its tile; this thread's rows of the block: mf, mf + 8
        bool ok = true;
        int j = 0, seg = 0;
        float row_mul[2];                                          // one over the power of two that a query row was laid out under
        bool scaled = false;                                       // ... is not one for some row of the warp
        const bool whole_blocks = c.block >= TN;
        // Query rows of a row block as K-major fp16 operands, by the warp that will hold their results.  (The products that read the rows before have ended:
        // the warp has seen the scores of the last tile.)  bfloat16 rows far from fp16's range under a power of two.
        auto lay_out = [&](const Segment& sg) -> bool {
            const int heads_here = min(HPG, c.G - sg.hg * HPG);
            auto valid = [&](int m) { return (m & (p.GP - 1)) < heads_here && sg.tq0 + q * p.QT + (m >> gp_bits) < c.Tq; };
            const bool some = __any_sync(0xffffffffu, valid(m0 + (lane & 15)));
            row_mul[0] = row_mul[1] = 1.f;
            scaled = false;
            if (some) {
                const int gl = p.lane0 + sg.lane_c, b = gl / c.Hkv, h0 = (gl - b * c.Hkv) * c.G + sg.hg * HPG;
                const uint16_t* src = static_cast<const uint16_t*>(c.q) + b * c.q_sb + int64_t(h0) * c.q_sh + int64_t(sg.tq0 + q * p.QT) * c.q_st;
                constexpr int CPR = D / 8;                         // 16-byte chunks of a row
                uint4 both[2][CPR / 4];                            // eight rows at a time: a row's chunks sit with neighbouring lanes of one load
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int u = 0; u < CPR / 4; ++u) {            // lane = row 8 e + (lane >> 2), chunk 4 u + (lane & 3)
                        const int m = m0 + 8 * e + (lane >> 2);
                        both[e][u] = make_uint4(0u, 0u, 0u, 0u);
                        if (valid(m)) both[e][u] = *reinterpret_cast<const uint4*>(src + (m & (p.GP - 1)) * c.q_sh + int64_t(m >> gp_bits) * c.q_st + (4 * u + (lane & 3)) * 8);
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r0 = 8 * e;
                    uint4 (&x)[CPR / 4] = both[e];
                    if (c.dtype == TQ_BF16) {
                        uint32_t mx = 0;
#pragma unroll
                        for (int u = 0; u < CPR / 4; ++u) mx = max(mx, largest16(x[u]));
                        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float big = __uint_as_float(mx << 16);
                        const float f = big >= 0.0078125f && big < 32768.f ? 1.f : stage_scale(mx << 16);
#pragma unroll
                        for (int u = 0; u < CPR / 4; ++u) x[u] = bf_to_half(x[u], f);
                        row_mul[e] = 1.f / f;
                        scaled = scaled || __any_sync(0xffffffffu, f != 1.f);
                    }
#pragma unroll
                    for (int u = 0; u < CPR / 4; ++u) {
                        const int r = m0 + r0 + (lane >> 2), ch = 4 * u + (lane & 3);
                        *reinterpret_cast<uint4*>(smem + P::OFF_Q + q * P::Q_TILE + (ch >> 3) * P::QBLK + r * 128 + (((ch ^ r) & 7) << 4)) = x[u];
                    }
                }
                fence_proxy_async();
            }
            mbar_arrive(bar(Q_FULL + q));
            return some;
        };
        int n = 0, tile_tok = 0;                                   // key tiles of the row block; the tile's first query token
        bool some = false;
        auto enter = [&](int job) {
            const Segment sg = segment(job);
            n = uniform(sg.n);
            tile_tok = uniform(sg.tq0 + q * p.QT);
            some = lay_out(sg);
        };
        enter(from.job);
        for (int job = from.job; job <= last_job && ok; ++job, ++seg) {
            if (!some) {
                // a warp without a row: the others' exponentials have the pipe to themselves.  (What it leaves in tensor memory meets rows that nobody reads.  A
                // score buffer is full again only behind the products that every warp of the query tile has arrived for, so that no arrival is a phase early.)
                for (int i = 0; i < n && ok; ++i, ++j) {
                    ok = __all_sync(0xffffffffu, wait_bar(SC_FULL + j % NSC, j / NSC) && wait_bar(S_FULL + sbuf(q, j), sph(j)));
                    if (!ok) break;
                    mbar_arrive(bar(P_FULL + sbuf(q, j)));
                    mbar_arrive(bar(SC_FREE + j % NSC));
                }
                if (job < last_job && ok) enter(job + 1);
                continue;
            }
            const int tile_first = q_pos0 + tile_tok, tile_lo = tile_first + p.QT - c.window;      // position of the tile's first row; the first token that its last row's window holds
            int pos[2];
            {
                const int hg = job / p.n_blk % p.HG, heads_here = min(HPG, c.G - hg * HPG);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int m = m0 + (lane >> 2) + 8 * k, tok = tile_tok + (m >> gp_bits);
                    pos[k] = (m & (p.GP - 1)) < heads_here && tok < c.Tq ? q_pos0 + tok : -1;
                }
            }
            // A row that has seen no token yet keeps m_ref = -1e30, has lvsc for a bias and asks for a reference at its first one.
            float vsc = 1.f, vthr = 0.f, lvsc = 0.f;               // (vthr 0: the first tile with a non-zero value scale picks the scale); log2(vsc)
            float m_ref[2] = {-1e30f, -1e30f}, bias[2] = {0.f, 0.f};       // bias = log2(vsc) - reference
            float thr[2] = {pos[0] >= 0 ? -1.f : INFINITY, pos[1] >= 0 ? -1.f : INFINITY};       // a tile's sum above this asks for another reference; a row's first tile always does
            u64 l2[2] = {pk(0.f, 0.f), pk(0.f, 0.f)};              // this thread's share of the rows' sums
            for (int i = 0; i < n; ++i, ++j) {
                const int s = j % NSC;
                {
                    const uint32_t sc_bar = bar(SC_FULL + s), s_bar = bar(S_FULL + sbuf(q, j)), sc_par = uint32_t(j / NSC) & 1u, s_par = uint32_t(sph(j)) & 1u;
                    if (!__all_sync(0xffffffffu, mbar_try(s_bar, s_par) && mbar_try(sc_bar, sc_par))) {
                        ok = wait_bar(S_FULL + sbuf(q, j), sph(j)) && wait_bar(SC_FULL + s, j / NSC);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    }
                }
                tc_fence_after();
                const float* sc = reinterpret_cast<const float*>(smem + P::OFF_SC + s * P::SC);
                const int2 at_end = *reinterpret_cast<const int2*>(sc + 2 * TN);
                const int base = at_end.x, end = at_end.y;         // (the tile's tokens lie before `end`)
                const float *kn = sc + t2, *vn = kn + TN;
                const bool one = whole_blocks && end == c.n8;      // the tile's tokens share a block, and its scales
                const uint32_t s_col = t_frag + sbuf(q, j) * TN;
                constexpr int NR = TN / 8;
                uint32_t v[4 * NR];                                // of eight columns: two of row g, two of row g + 8
                tmem_ld_frag64(s_col, v);
                const float k1 = sc[0], v1 = sc[TN];
                u64 nv[NR];
                if (!one) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) nv[r] = *reinterpret_cast<const u64*>(kn + 8 * r);
                }
                tmem_ld_wait();
                if (scaled) {
#pragma unroll
                    for (int r = 0; r < 4 * NR; ++r) v[r] = __float_as_uint(__uint_as_float(v[r]) * row_mul[(r >> 1) & 1]);
                }
                // t = score * key scale - reference + log2(value scale)
                auto place = [&](auto scale_of) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t* x = v + 2 * k;
                        const u64 b2 = pk(bias[k], bias[k]);
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            float x0, x1;
                            upk(fma2(pk(__uint_as_float(x[4 * r]), __uint_as_float(x[4 * r + 1])), scale_of(r), b2), x0, x1);
                            x[4 * r] = __float_as_uint(x0); x[4 * r + 1] = __float_as_uint(x1);
                        }
                    }
                };
                if (one) place([&](int) { return pk(k1, k1); });
                else place([&](int r) { return nv[r]; });
                if (base + TN - 1 > min(tile_first, end - 1) || (base < tile_lo && base + TN > c.sinks)) {      // some token of the tile is hidden from some row
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t* x = v + 2 * k;
                        const int hi = min(pos[k], end - 1) - base - t2, lo = pos[k] - c.window + 1 - base - t2, sk = c.sinks - base - t2;
#pragma unroll
                        for (int r = 0; r < 2 * NR; ++r) {
                            const int at = 8 * (r >> 1) + (r & 1);
                            if (at > hi || (at < lo && at >= sk)) x[4 * (r >> 1) + (r & 1)] = 0xff800000u;
                        }
                    }
                }
                // Weights, their sums, P = weight * value scale (both carry vsc) as fp16.  A row needs another reference when a weight exceeds
                // 2^SLACK, which its sum then does too: the sums are looked at behind the exponentials and no maximum is taken in the common case.
                // The lanes share the check of the tile's value scales, eight tokens' pairs each.
                float vmax = v1;
                if (!one) {
                    const float2 v2 = *reinterpret_cast<const float2*>(vn + 8 * g);
                    vmax = fmaxf(v2.x, v2.y);
#pragma unroll
                    for (int r = 0; r < NR; ++r) nv[r] = *reinterpret_cast<const u64*>(vn + 8 * r);
                }
                uint32_t w[2 * NR], rest[FINE ? 2 * NR : 1];       // the weights as fp16, and what that leaves
                u64 ls[2];
                auto weigh = [&](auto scale_of, auto sharing) {
                    ls[0] = ls[1] = pk(0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float y0 = __uint_as_float(v[4 * r + 2 * k]), y1 = __uint_as_float(v[4 * r + 2 * k + 1]);
                            const u64 x = decltype(sharing)::value && r % POLY_EVERY == POLY_EVERY - 1 ? ex2_by_fma(y0, y1) : pk(ex2(y0), ex2(y1));
                            ls[k] = add2(ls[k], x);
                            float x0, x1;
                            upk(mul2(x, scale_of(r)), x0, x1);
                            const __half2 h = __floats2half2_rn(x0, x1);
                            w[2 * r + k] = *reinterpret_cast<const uint32_t*>(&h);
                            if constexpr (FINE) {
                                const float2 hf = __half22float2(h);
                                rest[2 * r + k] = pack_h2(x0 - hf.x, x1 - hf.y);
                            }
                        }
                };
#pragma unroll 1
                for (int pass = 0;; ++pass) {
                    if (one) weigh([&](int) { return pk(v1, v1); }, std::bool_constant<NQ == 2>{});      // (of every token that is not finite, the other columns' sums tell)
                    else weigh([&](int r) { return nv[r]; }, std::false_type{});
                    bool again = vmax > vthr;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x0, x1;
                        upk(ls[k], x0, x1);
                        again = again || x0 + x1 > thr[k];
                    }
                    if (pass > 0 || !__any_sync(0xffffffffu, again)) break;
                    // Reference maximum / value scale: refreshed for the whole warp when any row needs it (rare after the first tile):
                    // the rows' sums and their O in tensor memory are rescaled.
                    float a[2], mx[2] = {-INFINITY, -INFINITY}, ratio = 1.f;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
#pragma unroll
                        for (int r = 0; r < NR; ++r) mx[k] = fmaxf(fmaxf(mx[k], __uint_as_float(v[4 * r + 2 * k])), __uint_as_float(v[4 * r + 2 * k + 1]));
#pragma unroll
                        for (int off = 1; off < 4; off <<= 1) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], off));
                    }
#pragma unroll
                    for (int off = 16; off; off >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, off));
                    if (vmax > vthr) {
                        int eb = (__float_as_int(vmax) >> 23) & 0xff;
                        eb = min(max(eb, 16), 240);
                        const float nsc = __int_as_float((254 + VS_LOG2 - eb) << 23);      // the largest value scale lands in [2^VS_LOG2, twice that)
                        ratio = nsc / vsc;
                        vsc = nsc;
                        vthr = VS_CAP / nsc;
                        lvsc = float(127 + VS_LOG2 - eb);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float mn = fmaxf(fmaxf(m_ref[k], mx[k] - bias[k]), -1e30f);
                        a[k] = ex2(m_ref[k] - mn) * ratio;
                        m_ref[k] = mn;
                        const float moved = mn > -1e30f ? lvsc - mn : lvsc, delta = moved - bias[k];
                        bias[k] = moved;
                        if (mn > -1e30f) thr[k] = float(1 << SLACK) * vsc;
                        l2[k] = mul2(l2[k], pk(a[k], a[k]));
                        uint32_t* x = v + 2 * k;
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            x[4 * r] = __float_as_uint(__uint_as_float(x[4 * r]) + delta);
                            x[4 * r + 1] = __float_as_uint(__uint_as_float(x[4 * r + 1]) + delta);
                        }
                    }
                    if (i > 0) {
                        ok = wait_bar(O_DONE + q, j - 1);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll 1
                        for (int c0 = 0; c0 < DP; c0 += 32) {
                            uint32_t o[16];
                            tmem_ld_frag32(t_frag + P::COL_O + q * DP + c0, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * a[(x >> 1) & 1]);
                            tmem_st_frag32(t_frag + P::COL_O + q * DP + c0, o);
                        }
                        tmem_st_wait();
                    }
                }
                if (!ok) break;
                l2[0] = add2(l2[0], ls[0]);
                l2[1] = add2(l2[1], ls[1]);
                tmem_st_half64(s_col, w);
                if constexpr (FINE) tmem_st_half64(s_col + TN / 2, rest);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(bar(P_FULL + sbuf(q, j)));
                mbar_arrive(bar(SC_FREE + s));
            }
            if (!ok) break;
            // ---- the next row block's queries, then this one's results, still as fragments: 32 bytes of a row from four lanes
            const int now_tok = tile_tok;
            if (job < last_job) enter(job + 1);
            float l_sum[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float l1;
                upk(l2[k], l_sum[k], l1);
                l_sum[k] += l1;
#pragma unroll
                for (int off = 1; off < 4; off <<= 1) l_sum[k] += __shfl_xor_sync(0xffffffffu, l_sum[k], off);
            }
            ok = __all_sync(0xffffffffu, wait_bar(ALL_DONE + q, seg));
            if (!ok) break;
            tc_fence_after();
            const int y = job / p.n_blk, lane_c = y / p.HG, gl = p.lane0 + lane_c, b = gl / c.Hkv, h0 = (gl - b * c.Hkv) * c.G + (y - lane_c * p.HG) * HPG;
            const bool parts = (job == from.job && from.tile > 0) || job == to.job;      // (a run that ends inside this row block, or began there)
            float* const part = p.part + (int64_t(blockIdx.x) * 2 + (seg > 0 ? 1 : 0)) * (P::ROWS * (D + 4)) + int64_t(mf) * (D + 4);
            if (parts && t2 == 0) {
#pragma unroll
                for (int k = 0; k < 2; ++k) *reinterpret_cast<float2*>(part + k * 8 * (D + 4) + D) = make_float2(m_ref[k] - lvsc, l_sum[k]);
            }
            const bool f16 = c.dtype == TQ_F16, odd = (t2 & 2) != 0;
            float il[2];
            bool store[2];
            char* dst[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int m = m0 + (lane >> 2) + 8 * k;
                il[k] = parts ? 1.f : 1.f / l_sum[k];
                store[k] = parts || pos[k] >= 0;
                dst[k] = parts ? reinterpret_cast<char*>(part + k * 8 * (D + 4) + t2)
                               : static_cast<char*>(c.out) + 2 * (((int64_t(b) * c.Hq + h0 + (m & (p.GP - 1))) * c.Tq + now_tok + (m >> gp_bits)) * D + (t2 & 4) + (odd ? 8 : 0));
            }
            auto rows = [&](int c0, uint32_t (&o)[16]) {           // of eight columns: two of row g, two of row g + 8
                tmem_ld_frag32(t_frag + P::COL_O + q * DP + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * il[(x >> 1) & 1]);
            };
            if (parts) {
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[16];
                    rows(c0, o);
#pragma unroll
                    for (int x = 0; x < 16; x += 2) *reinterpret_cast<uint2*>(dst[(x >> 1) & 1] + 4 * c0 + 8 * (x & 12)) = make_uint2(o[x], o[x + 1]);
                }
            } else {
                // two neighbouring lanes trade words: four columns each, the even one of eight columns, the odd one of the next eight
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[16];
                    rows(c0, o);
#pragma unroll
                    for (int x = 0; x < 16; x += 2) {
                        const float y = __uint_as_float(o[x]), z = __uint_as_float(o[x + 1]);
                        o[x] = f16 ? pack_h2(y, z) : pack_bf2(y, z);
                    }
#pragma unroll
                    for (int x = 0; x < 16; x += (x & 2) ? 6 : 2) {
                        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? o[x] : o[x + 4], 1);
                        if (store[(x >> 1) & 1]) *reinterpret_cast<uint2*>(dst[(x >> 1) & 1] + 2 * c0 + 4 * (x & 12)) = odd ? make_uint2(other, o[x + 4]) : make_uint2(o[x], other);
                    }
                }
            }
            tc_fence_before();                                     // (the next row block's products overwrite what was read here)
        }
    }
    // ---------------- teardown: every loop above is bounded, so every thread gets here ----------------
    tc_fence_before();
    __syncthreads();
    if (warp == P::SW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// A CTA per (cache lane, key tile of the call): its keys and values as operand tiles, its tokens' scales.  Bound by writing four bytes a code read.
constexpr int EX_T = 256;
template <int D> __global__ void __launch_bounds__(EX_T) blocks_fa_expand_kernel(const __grid_constant__ Params p) {
    constexpr uint32_t K_TILE = Plan<D, false>::K_TILE;
    constexpr int PIECES = TN * D / 16;                    // of a side
    const BlockAttendParams& c = p.a;
    const int lane_c = blockIdx.x / p.all.n, ord = blockIdx.x - lane_c * p.all.n, tid = threadIdx.x;
    const int64_t lane = p.lane0 + lane_c, at = int64_t(lane_c) * p.all.n + ord;
    const int base = (p.all.is_tail(ord) ? c.n8 : 0) + p.all.tile_of(ord) * TN;
    unsigned char* tiles = const_cast<unsigned char*>(p.tiles) + at * 2 * K_TILE;
    float* scales = const_cast<float*>(p.scales) + at * TILE_INFO;
    pdl_wait();                                            // (the tiles' memory may be what the kernel in front still reads or writes)
    if (tid == 0) *reinterpret_cast<int2*>(scales + 2 * TN) = make_int2(base, p.all.is_tail(ord) ? c.total : c.n8);
    if (!p.all.is_tail(ord)) {
        constexpr int U = 2 * PIECES / EX_T;               // (1024 / 16 = 64 tokens x D / 16 pieces x 2: a multiple of 256 for every D)
        static_assert(2 * PIECES % EX_T == 0, "pieces");
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = tid + u * EX_T, side = i >= PIECES, x = i - side * PIECES, row = x / (D / 16);
            raw[u] = make_uint4(0u, 0u, 0u, 0u);
            if (base + row < c.n8) ld_codes(raw[u], (side ? c.vc : c.kc) + ((lane * c.cap + base) * D + x * 16));
        }
        if (tid < TN) {
            const int tok = base + tid;
            float ks = 0.f, vs = 0.f;
            if (tok < c.n8) {
                ks = c.ks[lane * (c.cap >> c.shift) + (tok >> c.shift)] * c.scale_log2;
                vs = c.vs[lane * (c.cap >> c.shift) + (tok >> c.shift)];
                if (!finite_scale(vs)) { ks = __uint_as_float(0x7fffffffu); vs = 0.f; }
            }
            scales[tid] = ks;
            scales[TN + tid] = vs;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = tid + u * EX_T, side = i >= PIECES, x = i - side * PIECES, row = x / (D / 16), cc = x - row * (D / 16);
            uint4 lo, hi;
            expand16(raw[u], c.e4m3, lo, hi);
            unsigned char* dst = tiles + side * K_TILE;
            *reinterpret_cast<uint4*>(dst + chunk_place(row, 2 * cc)) = lo;
            *reinterpret_cast<uint4*>(dst + chunk_place(row, 2 * cc + 1)) = hi;
        }
    } else {
        // a warp per token, four at a time
        const int lane_t = tid & 31;
        const bool bf = c.dtype == TQ_BF16, mine = lane_t < D / 8;
        for (int r0 = tid >> 5; r0 < TN; r0 += 4 * EX_T / 32) {
            uint4 k[4], v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int tok = base + r0 + u * (EX_T / 32);
                k[u] = v[u] = make_uint4(0u, 0u, 0u, 0u);
                if (tok < c.total && mine) {
                    const int64_t src = (lane * c.block + (tok - c.n8)) * D + lane_t * 8;
                    k[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.kt) + src);
                    v[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.vt) + src);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * (EX_T / 32);
                const bool in = base + r < c.total;
                const uint32_t mk = __reduce_max_sync(0xffffffffu, largest16(k[u])), mv = __reduce_max_sync(0xffffffffu, largest16(v[u]));
                const bool fine = mv < (bf ? 0x7f80u : 0x7c00u);
                const float fk = bf ? stage_scale(mk << 16) : 1.f, fv = bf ? stage_scale(mv << 16) : 1.f;
                if (bf) { k[u] = bf_to_half(k[u], fk); v[u] = bf_to_half(v[u], fv); }
                if (!fine) v[u] = make_uint4(0u, 0u, 0u, 0u);
                if (mine) {
                    *reinterpret_cast<uint4*>(tiles + chunk_place(r, lane_t)) = k[u];
                    *reinterpret_cast<uint4*>(tiles + K_TILE + chunk_place(r, lane_t)) = v[u];
                }
                if (lane_t == 0) {
                    scales[r] = !in ? 0.f : fine ? c.scale_log2 / fk : __uint_as_float(0x7fffffffu);
                    scales[TN + r] = in && fine ? 1.f / fv : 0.f;
                }
            }
        }
    }
}

// Row blocks that several CTAs worked on: a warp per row adds their partials up in the CTAs' order.  Block = (boundary between two CTAs, eight rows); the block whose
// boundary is the row block's first one works.
template <int D, bool FUSED> __global__ void __launch_bounds__(256) blocks_fa_merge_kernel(const __grid_constant__ Params p) {
    using P = Plan<D, FUSED>;
    constexpr int NV = D / 32, GROUPS = P::ROWS / 8;
    const BlockAttendParams& c = p.a;
    const int lane = threadIdx.x & 31, edge = 1 + blockIdx.x / GROUPS, m = (blockIdx.x % GROUPS) * 8 + (threadIdx.x >> 5);
    const Params::Start s = p.start[edge], before = p.start[edge - 1];
    if (s.tile == 0 || (before.job == s.job && before.tile > 0)) return;
    const int y = s.job / p.n_blk, blk = s.job - y * p.n_blk, lane_c = y / p.HG, hg = y - lane_c * p.HG, gl = p.lane0 + lane_c, b = gl / c.Hkv, hkv = gl - b * c.Hkv;
    const int tok = blk * P::NQ * p.QT + (m >> 7) * p.QT + (m & 127) / p.GP, hh = (m & 127) % p.GP;
    if (hh >= min(HPG, c.G - hg * HPG) || tok >= c.Tq) return;
    pdl_wait();
    int last = edge;                                       // pieces: CTA edge - 1, edge, ..., last
    while (last + 1 < p.ctas && p.start[last + 1].job == s.job) ++last;
    const int first_slot = before.job == s.job ? 0 : 1;    // (the CTA in front has worked on another row block before)
    float x[NV], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = 0.f;
    for (int i = edge - 1; i <= last; ++i) {
        const float* part = p.part + (int64_t(i) * 2 + (i == edge - 1 ? first_slot : 0)) * (P::ROWS * (D + 4)) + int64_t(m) * (D + 4);
        const float2 ml = *reinterpret_cast<const float2*>(part + D);
        const float mn = fmaxf(fmaxf(top, ml.x), -1e30f), a = ex2(top - mn), w = ex2(ml.x - mn);
        top = mn;
        sum = sum * a + ml.y * w;
#pragma unroll
        for (int k = 0; k < NV; ++k) x[k] = x[k] * a + part[k * 32 + lane] * w;
    }
    const int64_t out = ((int64_t(b) * c.Hq + hkv * c.G + hg * HPG + hh) * c.Tq + tok) * D + lane;
    const float il = 1.f / sum;
#pragma unroll
    for (int k = 0; k < NV; ++k) store_from_f32(c.out, c.dtype, out + k * 32, x[k] * il);
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }

// How a call is laid out: row blocks, and in the workspace the partials, then (expanded) tiles and scales of `chunk` cache lanes at a time
constexpr size_t WS_CAP = size_t(1) << 29;
struct Layout { int HG, GP, QT, n_blk, chunk, ctas; Tiles all; size_t tiles, scales, bytes; int more; };      // more: rounds that want of room adds
template <int D, bool FUSED> Layout layout_of(const BlockAttendParams& p) {
    using P = Plan<D, FUSED>;
    const int g = std::min(p.G, HPG), lanes = p.B * p.Hkv;
    Layout l{(p.G + HPG - 1) / HPG, g <= 1 ? 1 : g <= 2 ? 2 : g <= 4 ? 4 : 8, 0, 0, lanes, 0, Tiles(p, p.total - p.Tq, p.total - 1), 0, 0, 0, 0};
    l.QT = TM / l.GP;
    l.n_blk = (p.Tq + P::NQ * l.QT - 1) / (P::NQ * l.QT);
    const int sms = std::min(blocks_sm_count(), MAX_CTAS);
    const size_t lane_tiles = size_t(l.all.n) * 2 * P::K_TILE, lane_scales = size_t(l.all.n) * P::SC;
    auto set = [&]() {
        l.ctas = int(std::min<int64_t>(sms, int64_t(l.chunk) * l.HG * l.n_blk * l.all.n));
        l.tiles = up(size_t(l.ctas) * 2 * P::ROWS * (D + 4) * sizeof(float));
        l.scales = l.tiles + (FUSED ? 0 : up(l.chunk * lane_tiles));
        l.bytes = l.scales + (FUSED ? 0 : up(l.chunk * lane_scales));
    };
    if (!FUSED)
        while (l.chunk > 1 && size_t(l.chunk) * (lane_tiles + lane_scales) > WS_CAP) l.chunk = (l.chunk + 1) / 2;
    const int chunk = l.chunk;
    for (set(); !FUSED && l.chunk > 1 && l.bytes > p.room; set()) l.chunk = (l.chunk + 1) / 2;
    l.more = (lanes + l.chunk - 1) / l.chunk - (lanes + chunk - 1) / chunk;
    return l;
}

// Runs of key tiles for the CTAs: where each one starts in the sequence of row blocks.  The row blocks of every (lane, head group) have the same tiles.  Either equal
// runs, wherever that cuts a row block, or runs of whole row blocks.  A cut costs partials and their merge: 5 us and, where every CTA of 148 has two of 256 rows, d = 128,
// 40 MB, 18 more; whole row blocks cost what the longest run has more than the others, a tile 1 us (fused) or 1.3 (two query tiles).
template <int D, bool FUSED> void divide(Params& p, int lanes) {
    const BlockAttendParams& a = p.a;
    const int rows = Plan<D, FUSED>::NQ * p.QT, q0 = a.total - a.Tq;
    auto tiles_of = [&](int blk) { return Tiles(a, q0 + blk * rows, q0 + std::min((blk + 1) * rows, a.Tq) - 1).n; };
    int64_t per_y = 0;
    for (int i = 0; i < p.n_blk; ++i) per_y += tiles_of(i);
    const int64_t total = per_y * lanes * p.HG;
    const int64_t jobs = int64_t(lanes) * p.HG * p.n_blk;
    const int ctas = p.ctas, most = int(std::max<int64_t>(1, std::min<int64_t>(ctas, total / 4)));      // (cut: at least four tiles a CTA: a partial more to join costs about as much)
    auto fill = [&](bool whole) -> int64_t {               // -> tiles of the longest run
        int blk = 0, n = 0;
        int64_t y = 0, before = 0, longest = 0, last = 0;  // tiles in front of row block `blk` of y
        p.start[0] = Params::Start{0, 0};
        const int want = whole ? ctas : most;
        for (int i = 1; i <= want; ++i) {
            int64_t at = total * i / want;
            const int64_t ny = i == want ? int64_t(lanes) * p.HG : at / per_y, off = at - ny * per_y;
            if (ny != y) { y = ny; blk = 0; before = 0; }
            while (blk < p.n_blk && before + tiles_of(blk) <= off) before += tiles_of(blk++);
            Params::Start s{int(y * p.n_blk + blk), int(off - before)};
            if (whole && s.tile > 0) {                     // to the nearer end of the row block
                const bool next = 2 * s.tile > tiles_of(blk);
                at += (next ? tiles_of(blk) : 0) - s.tile;
                s = Params::Start{s.job + (next ? 1 : 0), 0};
            }
            if (s.job == p.start[n].job && s.tile == p.start[n].tile) continue;        // (no run is empty)
            longest = std::max(longest, at - last);
            last = at;
            p.start[++n] = s;
        }
        p.ctas = n;
        return longest;
    };
    int64_t whole = 0;                                     // tiles of the longest run of whole row blocks
    if (jobs <= ctas) {                                    // a CTA each (64 row blocks of two tiles: 17 us as runs of four)
        for (int i = 0; i < p.n_blk; ++i) whole = std::max<int64_t>(whole, tiles_of(i));
        for (int i = 0; i <= int(jobs); ++i) p.start[i] = Params::Start{i, 0};
        p.ctas = int(jobs);
    } else {
        whole = fill(true);
    }
    const double cut_us = 5.0 + 0.45e-6 * double(most) * 2 * Plan<D, FUSED>::ROWS * (D + 4) * 4, tile_us = Plan<D, FUSED>::NQ == 1 ? 1.0 : 1.3;
    if (double(whole - (total + most - 1) / most) * tile_us > cut_us) fill(false);
}

Params params_of(const BlockAttendParams& a, const Layout& l, unsigned char* ws) {
    return Params{a, 0, l.HG, l.GP, l.QT, l.n_blk, l.ctas, {}, reinterpret_cast<float*>(ws), ws + l.tiles, reinterpret_cast<const float*>(ws + l.scales), l.all, nullptr};
}
bool cuts(const Params& p) {
    bool any = false;
    for (int i = 1; i < p.ctas; ++i) any = any || p.start[i].tile > 0;
    return any;
}

template <int D, bool FUSED> int launch(const BlockAttendParams& a, unsigned char* ws, cudaStream_t st) {
    using P = Plan<D, FUSED>;
    const Layout l = layout_of<D, FUSED>(a);
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    if (dev < 0 || dev >= 64 || !set[dev].load()) {
        cudaError_t e = cudaSuccess;
        for (auto* k : {blocks_fa_kernel<D, FUSED, false>, blocks_fa_kernel<D, FUSED, true>})
            if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::SMEM));
        if (e != cudaSuccess) return fail(TQ_ERR_LAUNCH, "tq_blocks_attend: shared memory %zu B: %s", P::SMEM, cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) set[dev].store(true);
    }
    Params p = params_of(a, l, ws);
    if (!(p.status = decode_status_ptr())) return fail(TQ_ERR_LAUNCH, "tq_blocks_attend: cannot locate the status word");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int lanes = a.B * a.Hkv;
    for (int lane0 = 0; lane0 < lanes; lane0 += l.chunk) {
        const int n = std::min(l.chunk, lanes - lane0);
        p.lane0 = lane0;
        p.ctas = l.ctas;
        divide<D, FUSED>(p, n);
        if (!FUSED) {
            cfg.gridDim = dim3(unsigned(int64_t(n) * l.all.n));
            cfg.blockDim = dim3(EX_T);
            cfg.dynamicSmemBytes = 0;
            cudaLaunchKernelEx(&cfg, blocks_fa_expand_kernel<D>, p);
            if (int rc = check_launch("tq_blocks_attend")) return rc;
        }
        cfg.gridDim = dim3(unsigned(p.ctas));
        cfg.blockDim = dim3(P::NT);
        cfg.dynamicSmemBytes = P::SMEM;
        cudaLaunchKernelEx(&cfg, a.dtype == TQ_F16 ? blocks_fa_kernel<D, FUSED, true> : blocks_fa_kernel<D, FUSED, false>, p);
        if (int rc = check_launch("tq_blocks_attend")) return rc;
        if (!cuts(p)) continue;
        cfg.gridDim = dim3(unsigned(p.ctas - 1) * (P::ROWS / 8));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        cudaLaunchKernelEx(&cfg, blocks_fa_merge_kernel<D, FUSED>, p);
        if (int rc = check_launch("tq_blocks_attend")) return rc;
    }
    return TQ_OK;
}

// What a call is expected to cost, in us, fitted to 300 calls (d = 64, 128 and 256; 8 to 128 lanes; 100 to 12,000 tokens; 16 to 1024 query rows a lane): set-up 7.7, a key
// tile of a CTA's run 1.3 (fused) or 1.1 at d = 128, a cut 3.2 and the partials' bytes, for expanded tiles another launch and six bytes a coordinate, read and written.
// Measured, fused / expanded, 4 heads on 1 at d = 128: 8 lanes x 12,000 tokens, 128 query rows a lane 36 / 52, 512 63 / 65, 1024 109 / 85; 64 lanes x 12,000, 256 rows
// 217 / 221, 384 322 / 296, 512 432 / 319; 64 lanes x 700, 256 22 / 32, 1024 67 / 48.
template <int D, bool FUSED> double cost(const BlockAttendParams& p) {
    const Layout l = layout_of<D, FUSED>(p);
    if (l.bytes > p.room) return 1e30;
    const int64_t lanes = int64_t(p.B) * p.Hkv, jobs = lanes * l.HG * l.n_blk, sms = blocks_sm_count();
    const int rows = Plan<D, FUSED>::NQ * l.QT;
    double n = 0;                                          // tiles of a row block, on the mean of the first and the last
    for (int blk : {0, l.n_blk - 1}) n += 0.5 * Tiles(p, p.total - p.Tq + blk * rows, p.total - p.Tq + std::min((blk + 1) * rows, p.Tq) - 1).n;
    const double tile = (FUSED ? 1.3 : 1.1) * (D <= 64 ? 0.7 : D <= 96 ? 0.85 : D <= 128 ? 1.0 : 0.86), runs = std::min(double(sms), double(jobs) * n / 4);
    const double whole = double((jobs + sms - 1) / sms) * n * tile, cut = std::max(4.0, double(jobs) * n / double(sms)) * tile + 3.2 + 4.6e-7 * runs * 2 * Plan<D, FUSED>::ROWS * (D + 4) * 4;
    return 7.7 + 12.0 * l.more + (runs < double(jobs) ? whole : std::min(whole, cut)) + (FUSED ? 0.0 : 4.0 + 2.1e-7 * double(lanes) * l.all.n * TN * 6 * D);
}
// Whether the codes are converted in the attention kernel (not at d = 256, where its eight converting warps cannot keep up: 3 times the other way's time).
template <int D> bool fused(const BlockAttendParams& p) {
    if constexpr (D > 128) return false;
    else return cost<D, true>(p) <= cost<D, false>(p);
}
template <int D> double least(const BlockAttendParams& p) {
    if constexpr (D > 128) return cost<D, false>(p);
    else return std::min(cost<D, true>(p), cost<D, false>(p));
}
template <int D> size_t workspace(const BlockAttendParams& p) {
    if constexpr (D <= 128)
        if (fused<D>(p)) return layout_of<D, true>(p).bytes;
    return layout_of<D, false>(p).bytes;
}
template <int D, bool FUSED> int choice(const BlockAttendParams& a) {
    const Layout l = layout_of<D, FUSED>(a);
    Params p = params_of(a, l, nullptr);
    divide<D, FUSED>(p, std::min(l.chunk, a.B * a.Hkv));
    return (FUSED ? TQ_BLOCKS_FUSED : TQ_BLOCKS_EXPANDED) + (cuts(p) ? 1 : 0);
}
template <int D> int choice_any(const BlockAttendParams& p) {
    if constexpr (D <= 128)
        if (fused<D>(p)) return choice<D, true>(p);
    return choice<D, false>(p);
}
template <int D> int launch_any(const BlockAttendParams& p, unsigned char* ws, cudaStream_t s) {
    if constexpr (D <= 128)
        if (fused<D>(p)) return launch<D, true>(p, ws, s);
    return launch<D, false>(p, ws, s);
}

}  // namespace bfa

// (fp16 tokens, whose second part costs 7 to 25% of this kernel, choose by the same figures: over 23 calls around the borders the choice was within 0.1% of the best on the mean, 2% at worst.)
// Whether this kernel takes the call rather than blocks_attend.cu's, which reads the codes once for every eight query rows of a lane.  us measured, that one / this one,
// 4 heads on 1 at d = 128: 8 lanes x 12,000 tokens, 32 rows a lane 25 / 34, 64 39 / 34, 128 66 / 36; 64 lanes x 12,000, 16 72 / 109, 32 131 / 130, 64 259 / 136; 64 lanes x 700,
// 32 17 / 21, 64 31 / 21; 64 lanes x 100, 32 9 / 10, 64 16 / 10, 128 30 / 10.  The choice among all the ways was within 0.7% of the best on the mean of the calls swept; the
// largest miss (58%, of 20 us) has d = 256.
bool blocks_fa_takes(const BlockAttendParams& p) {
    if (p.dtype == TQ_F32 || (p.D != 64 && p.D != 96 && p.D != 128 && p.D != 256) || p.kn != nullptr) return false;
    if (int64_t(p.Tq) * p.G <= HPG || int64_t(p.B) * p.Hkv * p.G * p.Tq >= (int64_t(1) << 29)) return false;
    const double us = p.D == 64 ? bfa::least<64>(p) : p.D == 96 ? bfa::least<96>(p) : p.D == 128 ? bfa::least<128>(p) : bfa::least<256>(p);
    return us < blocks_split_us(p);
}
size_t blocks_fa_workspace(const BlockAttendParams& p) {
    return p.D == 64 ? bfa::workspace<64>(p) : p.D == 96 ? bfa::workspace<96>(p) : p.D == 128 ? bfa::workspace<128>(p) : bfa::workspace<256>(p);
}
int blocks_fa_choice(const BlockAttendParams& p) {
    return p.D == 64 ? bfa::choice_any<64>(p) : p.D == 96 ? bfa::choice_any<96>(p) : p.D == 128 ? bfa::choice_any<128>(p) : bfa::choice_any<256>(p);
}
int launch_blocks_fa(const BlockAttendParams& p, cudaStream_t s) {
    unsigned char* ws = reinterpret_cast<unsigned char*>(p.part);
    if (p.D == 64) return bfa::launch_any<64>(p, ws, s);
    if (p.D == 96) return bfa::launch_any<96>(p, ws, s);
    if (p.D == 128) return bfa::launch_any<128>(p, ws, s);
    return bfa::launch_any<256>(p, ws, s);
}

}  // namespace tq
