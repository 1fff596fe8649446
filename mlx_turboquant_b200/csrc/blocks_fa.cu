// Causal attention of several query tokens over the 8-bit block cache, window and sinks included: flash attention on the fifth-generation tensor cores
// that expands the codes as it goes.
//
// Codes are exact as fp16, so a CTA turns a key tile of 64 tokens (and the value tile) into fp16 operands in shared memory once and multiplies them with
// up to 256 query rows; the blocks' scales stay float32 and meet the scores as a multiply-add and the softmax weights as a factor.  One launch, no
// expanded rows in global memory: the cache's bytes are read, a byte a value, by every CTA that needs them, mostly from L2.
//
// A CTA owns NQ (2; 1 at d = 256) tiles of 128 rows = 128 / GP query tokens x the GP query heads of a GQA group, and a range of the key tiles that some row
// sees: sinks, the window's blocks, the tail.
//   * four warps expand: two the keys, two the values; a thread's next 16-byte pieces of codes are on their way in registers while the tile before is used.
//     Rows of the tail (as they came) under a power of two each when they are bfloat16;
//   * 8 NQ softmax warps, two rows' shares per thread: tcgen05.ld of the scores as fragments, one packed multiply-add each, ex2, P (fp16) back into tensor
//     memory; a row's reference maximum is looked at through its sum;
//   * one warp issues S = Q K^T and O += P V, the two query tiles alternating, scores two key tiles ahead.
// blocks_fa_merge_kernel joins the partials of rows whose key tiles were split over several CTAs, in their order.
//
// Every mbarrier wait is bounded; one that runs out leaves status 114 (tq_device_status) and raises a flag that ends every other wait; products in flight
// are waited for (bounded), tensor memory is freed on every path.
#include <algorithm>
#include <atomic>

#include "blocks.cuh"
#include "fa_dev.cuh"

namespace tq {

int* decode_status_ptr();

namespace bfa {

using namespace fa;

constexpr int ERR_WAIT = 114;
constexpr int NSC = 8;                                 // tiles' scales in flight
constexpr int MAX_RANGES = 16;                         // key ranges of a row block

template <int D> struct Plan {
    static constexpr int NQ = D == 256 ? 1 : 2;        // query tiles per CTA
    static constexpr int TN = 64;                      // tokens per key tile
    static constexpr int SB = 2;                       // score buffers per query tile
    static constexpr int ST = D == 256 ? 2 : 4;        // key tiles (and value tiles) in shared memory
    static constexpr int NBLK = (D + 63) / 64;         // 64-column blocks of a row
    static constexpr int DP = NBLK * 64;               // columns of O (d = 96: nobody reads the last 32)
    static constexpr int SW = NQ * 8, XW = 4, NT = (SW + 1 + XW) * 32;       // softmax warps, the MMA warp, expanding warps
    static constexpr int CH = D / 16;                  // 16-byte pieces of a tile per expanding thread (64 a side)
    static constexpr uint32_t QBLK = TM * 128u, KBLK = TN * 128u;            // bytes of a 64-column block
    static constexpr uint32_t Q_TILE = NBLK * QBLK, K_TILE = NBLK * KBLK;
    static constexpr uint32_t OFF_Q = 0, OFF_K = NQ * Q_TILE, OFF_V = OFF_K + ST * K_TILE;
    static constexpr uint32_t SC = 2 * TN * 4 + 16, OFF_SC = OFF_V + ST * K_TILE;      // per tile float keys[TN], values[TN], 64 bits of spoilt tokens
    static constexpr uint32_t OFF_BAR = OFF_SC + NSC * SC;
    static constexpr uint32_t OFF_SLOT = OFF_BAR + 8 * 48;                   // [0] tensor-memory base, [1] abort, [2] largest query
    static constexpr size_t NEED = OFF_SLOT + 16 + 1024, SMEM = NEED > 116 * 1024 ? NEED : 116 * 1024;      // one CTA per SM: it takes all of the tensor memory
    static constexpr uint32_t COL_O = NQ * SB * TN;                          // scores first, then the accumulators
    static_assert(COL_O + NQ * DP <= 512, "tensor memory");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
enum Bars { K_FULL = 0, K_FREE = 4, V_FULL = 8, V_FREE = 12, SC_FULL = 16, SC_FREE = 24, S_FULL = 32, P_FULL = 36, O_DONE = 40, ALL_DONE = 42, DRAIN = 44 };       // (45 of 8 bytes)

struct Params {
    BlockAttendParams a;
    int HG, GP, QT;                                    // head groups, padded heads of one; query tokens per query tile
    int n_blk, n_splits;                               // row blocks, key ranges
    float* part;                                       // (lane x head group, row block, range, NQ * 128 rows, D + 4)
    int* status;
};

template <int D>
__global__ void __launch_bounds__(Plan<D>::NT, 1) blocks_fa_kernel(const __grid_constant__ Params p) {
    using P = Plan<D>;
    constexpr int NQ = P::NQ, TN = P::TN, DP = P::DP;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t raw_addr = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t sbase = (raw_addr + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (sbase - raw_addr);
    volatile uint32_t* slot = reinterpret_cast<volatile uint32_t*>(smem + P::OFF_SLOT);
    auto bar = [&](int which) -> uint32_t { return sbase + P::OFF_BAR + 8u * uint32_t(which); };
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // (uniform)
    const BlockAttendParams& c = p.a;

    // CTA = (lane x head group, row block, key range); the latest query rows (the longest runs of tiles) first
    const int y = blockIdx.x / (p.n_blk * p.n_splits), x_of = blockIdx.x - y * p.n_blk * p.n_splits;
    const int blk = p.n_blk - 1 - x_of / p.n_splits, split = x_of % p.n_splits;
    const int lane_c = y / p.HG, hg = y - lane_c * p.HG, b = lane_c / c.Hkv, hkv = lane_c - b * c.Hkv;
    const int heads_here = min(HPG, c.G - hg * HPG);
    const int tq0 = blk * NQ * p.QT, gp_bits = 31 - __clz(p.GP);
    auto row_head = [&](int m) { return m & (p.GP - 1); };
    auto row_token = [&](int m) { return tq0 + (m >> 7) * p.QT + ((m & 127) >> gp_bits); };
    auto row_valid = [&](int m) { return row_head(m) < heads_here && row_token(m) < c.Tq; };
    auto row_out = [&](int m) -> int64_t { return ((int64_t(b) * c.Hq + hkv * c.G + hg * HPG + row_head(m)) * c.Tq + row_token(m)) * D; };
    // key tiles of this CTA: its share of those that some row of it sees - sinks, the window's in blocks, the tail's
    const int q_pos0 = c.total - c.Tq, first_pos = q_pos0 + tq0, last_pos = q_pos0 + min(tq0 + NQ * p.QT, c.Tq) - 1;
    const int low = max(0, first_pos - c.window + 1), sinks = min(c.sinks, low), code_end = min(last_pos + 1, c.n8);
    const int low_tile = min(low, c.n8) / TN, n_win = low >= code_end ? 0 : (code_end + TN - 1) / TN - low_tile;
    const int sink_tiles = (min(sinks, code_end) + TN - 1) / TN, n_sink = n_win > 0 ? min(sink_tiles, low_tile) : sink_tiles;
    const int tail_tile = sinks > c.n8 ? 0 : max(low - c.n8, 0) / TN, n_tail = last_pos < c.n8 ? 0 : (last_pos + 1 - c.n8 + TN - 1) / TN - tail_tile;
    const int n_code = n_sink + n_win, n_all = n_code + n_tail;
    const int per = (n_all + p.n_splits - 1) / p.n_splits, t_lo = split * per, n = max(0, min(t_lo + per, n_all) - t_lo);
    auto is_tail = [&](int j) { return t_lo + j >= n_code; };
    auto tile_base = [&](int j) {                                          // first token of key tile j
        const int t = t_lo + j;
        return t < n_sink ? t * TN : t < n_code ? (low_tile + t - n_sink) * TN : c.n8 + (tail_tile + t - n_code) * TN;
    };

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(K_FULL + i), 64); mbar_init(bar(K_FREE + i), 1); mbar_init(bar(V_FULL + i), 64); mbar_init(bar(V_FREE + i), 1);
            mbar_init(bar(S_FULL + i), 1); mbar_init(bar(P_FULL + i), 256);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(O_DONE + i), 1); mbar_init(bar(ALL_DONE + i), 1); }
        mbar_init(bar(DRAIN), 1);
        for (int i = 0; i < NSC; ++i) { mbar_init(bar(SC_FULL + i), 128); mbar_init(bar(SC_FREE + i), NQ * 256); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        slot[1] = 0u;
        slot[2] = 0u;
    }
    if (warp == P::SW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + P::OFF_SLOT), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    if (p.n_splits > 1) pdl_trigger();
    // ---- the query rows as K-major fp16 operands; bfloat16 ones under one power of two that takes the CTA's largest element to [2^7, 2^8)
    // (what a smaller row loses then is 2^-33 of the largest score: scores enter the softmax by their differences)
    float mul = c.scale_log2;                                              // scale * log2(e) over that power: rides on the keys' scales
    {
        constexpr int N = NQ * TM * (D / 8), U = (N + P::NT - 1) / P::NT;
        uint4 x[U];
        uint32_t mx = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = tid + u * P::NT, m = i / (D / 8), c8 = i - m * (D / 8);
            x[u] = make_uint4(0u, 0u, 0u, 0u);
            if (i < N && row_valid(m)) {
                const uint16_t* src = static_cast<const uint16_t*>(c.q) + b * c.q_sb + int64_t(hkv * c.G + hg * HPG + row_head(m)) * c.q_sh + int64_t(row_token(m)) * c.q_st;
                x[u] = *reinterpret_cast<const uint4*>(src + c8 * 8);
            }
            const uint32_t k = 0x7fff7fffu, z = __vmaxu2(__vmaxu2(x[u].x & k, x[u].y & k), __vmaxu2(x[u].z & k, x[u].w & k));
            mx = max(mx, max(z & 0xffffu, z >> 16));
        }
        const bool bf = c.dtype == TQ_BF16;
        float f = 1.f;
        if (bf) {
            mx = __reduce_max_sync(0xffffffffu, mx);
            if (lane == 0) atomicMax(const_cast<uint32_t*>(slot + 2), mx << 16);
            __syncthreads();
            f = stage_scale(slot[2]);
            mul /= f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = tid + u * P::NT, m = i / (D / 8), c8 = i - m * (D / 8), r = m & 127;
            if (i >= N) continue;
            if (bf) {
                auto two = [&](uint32_t v) { return pack_h2(__uint_as_float(v << 16) * f, __uint_as_float(v & 0xffff0000u) * f); };
                x[u] = make_uint4(two(x[u].x), two(x[u].y), two(x[u].z), two(x[u].w));
            }
            *reinterpret_cast<uint4*>(smem + P::OFF_Q + (m >> 7) * P::Q_TILE + (c8 >> 3) * P::QBLK + r * 128 + (((c8 & 7) ^ (r & 7)) << 4)) = x[u];
        }
        fence_proxy_async();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, slot[0], 0);

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
    // products end (bounded) before their memory is given up, also after a wait that ran out
    auto drain = [&](int which, int phase) {
        for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try(bar(which), uint32_t(phase & 1)); ++i) {}
    };
    // score buffer of (query tile q, key tile j) and the phase of its barriers
    constexpr int SB = P::SB, ST = P::ST;
    auto sbuf = [](int q, int j) { return q * SB + j % SB; };
    auto sph = [](int j) { return j / SB; };
    auto first_row = [&]() { return (warp >> 3) * TM + (warp & 3) * 32 + (warp & 4) * 4 + (lane >> 2); };      // a softmax thread has this row and the eighth one after it

    if (warp > P::SW) {
        // ======================= codes to operands: two warps the keys, two the values =======================
        const int side = (warp - P::SW - 1) >> 1, ct = tid - (P::SW + 1 + 2 * side) * 32;                  // 0 ... 63
        const int64_t lane64 = lane_c;
        const uint8_t* codes = (side ? c.vc : c.kc) + lane64 * c.cap * D;
        const float* scales = (side ? c.vs : c.ks) + lane64 * (c.cap >> c.shift);
        const uint16_t* tail = static_cast<const uint16_t*>(side ? c.vt : c.kt) + lane64 * c.block * D;
        const uint32_t ring = sbase + (side ? P::OFF_V : P::OFF_K);
        const int full = side ? V_FULL : K_FULL, free_ = side ? V_FREE : K_FREE;
        const float factor = side ? 1.f : mul;
        uint4 raw[P::CH];
        float sc = 0.f;
        auto fetch = [&](int j, int u) {                                   // piece u of tile j (a multiple of 16 tokens of it are in blocks)
            const int i = ct + 64 * u, row = i / (D / 16);
            raw[u] = make_uint4(0u, 0u, 0u, 0u);
            const int tok = tile_base(j) + row;
            if (tok < c.n8) ld_codes(raw[u], codes + (int64_t(tok) * D + (i - row * (D / 16)) * 16));
        };
        auto fetch_scale = [&](int j) {
            const int tok = tile_base(j) + ct;
            sc = tok < c.n8 ? scales[tok >> c.shift] : 0.f;
        };
        if (n > 0 && !is_tail(0)) {
#pragma unroll
            for (int u = 0; u < P::CH; ++u) fetch(0, u);
            fetch_scale(0);
        }
        for (int j = 0; j < n; ++j) {
            const int st = j % ST, s = j % NSC;
            if (j >= ST && !__all_sync(0xffffffffu, wait_bar(free_ + st, j / ST - 1))) break;
            if (j >= NSC && !__all_sync(0xffffffffu, wait_bar(SC_FREE + s, j / NSC - 1))) break;
            const uint32_t tile = ring + st * P::K_TILE;
            float* scale_out = reinterpret_cast<float*>(smem + P::OFF_SC + s * P::SC) + side * TN + ct;
            float v = 0.f;
            bool spoilt = false;
            if (!is_tail(j)) {
                const bool more = j + 1 < n && !is_tail(j + 1);
                v = sc;
#pragma unroll
                for (int u = 0; u < P::CH; ++u) {
                    const int i = ct + 64 * u, row = i / (D / 16), cc = i - row * (D / 16);
                    uint4 lo, hi;
                    if (c.e4m3) {
                        halves<true>(raw[u].x, lo.x, lo.y); halves<true>(raw[u].y, lo.z, lo.w); halves<true>(raw[u].z, hi.x, hi.y); halves<true>(raw[u].w, hi.z, hi.w);
                    } else {
                        halves<false>(raw[u].x, lo.x, lo.y); halves<false>(raw[u].y, lo.z, lo.w); halves<false>(raw[u].z, hi.x, hi.y); halves<false>(raw[u].w, hi.z, hi.w);
                    }
                    // 16 columns are two chunks of 16 bytes of a row; every other group of four lanes writes its second one first: eight lanes, eight places
                    const bool swap = cc & 4;
                    const uint32_t at = tile + uint32_t(cc >> 2) * P::KBLK + uint32_t(row) * 128u, c0 = uint32_t(cc & 3) * 2u + (swap ? 1u : 0u), rx = uint32_t(row & 7);
                    st_shared(at + ((c0 ^ rx) << 4), swap ? hi : lo);
                    st_shared(at + (((c0 ^ 1u) ^ rx) << 4), swap ? lo : hi);
                    if (more) fetch(j + 1, u);
                }
                if (more) fetch_scale(j + 1);
            } else {
                // a thread per token: 16-bit rows, bfloat16 ones under their power of two
                const int tok = tile_base(j) + ct;
                const uint4* src = reinterpret_cast<const uint4*>(tail + int64_t(tok - c.n8) * D);
                const bool in = tok < c.total && tok <= last_pos, bf = c.dtype == TQ_BF16;
                uint32_t mx = 0;
                if (in)
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const uint4 x = src[i];
                        const uint32_t k = 0x7fff7fffu, z = __vmaxu2(__vmaxu2(x.x & k, x.y & k), __vmaxu2(x.z & k, x.w & k));
                        mx = max(mx, max(z & 0xffffu, z >> 16));
                    }
                const float f = bf ? stage_scale(mx << 16) : 1.f;
                // a value row that is not finite would reach rows that it is hidden from as 0 * inf: zeros, and the token marked
                spoilt = side && mx >= (bf ? 0x7f80u : 0x7c00u);
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (in && !spoilt) {
                        x = src[i];
                        if (bf) {
                            auto two = [&](uint32_t w) { return pack_h2(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f); };
                            x = make_uint4(two(x.x), two(x.y), two(x.z), two(x.w));
                        }
                    }
                    st_shared(tile + uint32_t(i >> 3) * P::KBLK + uint32_t(ct) * 128u + ((uint32_t(i & 7) ^ uint32_t(ct & 7)) << 4), x);
                }
                v = in ? 1.f / f : 0.f;
            }
            if (side) {
                spoilt = spoilt || !(fabsf(v) <= 3.4028235e38f);
                if (spoilt) v = 0.f;
                const uint32_t bits = __ballot_sync(0xffffffffu, spoilt);
                if (lane == 0) reinterpret_cast<uint32_t*>(smem + P::OFF_SC + s * P::SC + 2 * TN * 4)[ct >> 5] = bits;
            }
            *scale_out = v * factor;
            fence_proxy_async();
            mbar_arrive(bar(full + st));
            mbar_arrive(bar(SC_FULL + s));
        }
        __syncwarp();
    } else if (warp == P::SW) {
        // ======================= MMA issue: one warp, uniform =======================
        if (n > 0) {
            auto issue_qk = [&](int q, int j) {                    // S = Q K^T of key tile j
                const uint32_t s = tmem + sbuf(q, j) * TN;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(s, desc_k(sbase + P::OFF_Q + q * P::Q_TILE, P::QBLK, ks), desc_k(sbase + P::OFF_K + (j % ST) * P::K_TILE, P::KBLK, ks),
                            idesc_of(TN, false), ks > 0 ? 1u : 0u);
                umma_commit(bar(S_FULL + sbuf(q, j)));
            };
            auto issue_pv = [&](int q, int j) {                    // O += P V
                const uint32_t a = tmem + sbuf(q, j) * TN;
#pragma unroll
                for (int ks = 0; ks < TN / 16; ++ks)
                    umma_ts(tmem + P::COL_O + q * DP, a + ks * 8, desc_mn(sbase + P::OFF_V + (j % ST) * P::K_TILE, P::KBLK, ks), idesc_of(DP, true),
                            (j > 0 || ks > 0) ? 1u : 0u);
                umma_commit(bar(O_DONE + q));
                if (j == n - 1) umma_commit(bar(ALL_DONE + q));    // (a barrier of its own: a parity wait on O_DONE could be two phases early or one late)
            };
            auto wait_all = [&](int which, int phase) -> bool { return __all_sync(0xffffffffu, wait_bar(which, phase)); };
            bool ok = true;
            for (int j = 0; j < min(n, SB) && ok; ++j) {
                ok = wait_all(K_FULL + j % ST, j / ST);
                if (!ok) break;
                tc_fence_after();
                for (int q = 0; q < NQ; ++q) issue_qk(q, j);
                umma_commit(bar(K_FREE + j % ST));
            }
            for (int j = 0; j < n && ok; ++j) {
                ok = wait_all(V_FULL + j % ST, j / ST);
                const int jn = j + SB;                             // the key tile whose scores go where P of tile j sits now
                for (int q = 0; q < NQ && ok; ++q) {
                    ok = wait_all(P_FULL + sbuf(q, j), sph(j));
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(q, j);
                    if (q == NQ - 1) umma_commit(bar(V_FREE + j % ST));
                    if (jn < n) {                                  // (the tensor core takes one thread's products in order)
                        if (q == 0) ok = wait_all(K_FULL + jn % ST, jn / ST);
                        if (!ok) break;
                        tc_fence_after();
                        issue_qk(q, jn);
                        if (q == NQ - 1) umma_commit(bar(K_FREE + jn % ST));
                    }
                }
            }
            if (!ok) { umma_commit(bar(DRAIN)); drain(DRAIN, 0); }
        }
        __syncwarp();
    } else if (__any_sync(0xffffffffu, row_valid(first_row()) || row_valid(first_row() + 8))) {
        // ======================= softmax: two rows per thread, sixteen columns of each =======================
        // Scores are read as mma.sync fragments: lane 4 g + t of a warp holds columns 8 r + 2 t, + 1 of rows g and g + 8 of its sixteen.
        const int q = warp >> 3, hh = (warp >> 2) & 1, g = lane >> 2, t2 = 2 * (lane & 3);       // query tile; half of the 32 lanes
        const uint32_t t_frag = tmem + (uint32_t((warp & 3) * 32 + 16 * hh) << 16);
        const int mf = first_row();
        const int tile_first = q_pos0 + tq0 + q * p.QT, tile_lo = tile_first + p.QT - c.window;  // position of the tile's first row; the first token that its last row's window holds
        int pos[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) pos[k] = row_valid(mf + 8 * k) ? q_pos0 + row_token(mf + 8 * k) : -1;
        // A row that has seen no token yet keeps m_ref = -1e30, has lvsc for a bias and asks for a reference at its first one.
        float vsc = 1.f, vthr = 0.f, lvsc = 0.f;                   // (vthr 0: the first tile with a non-zero value scale picks the scale); log2(vsc)
        float m_ref[2] = {-1e30f, -1e30f};
        u64 l2[2] = {pk(0.f, 0.f), pk(0.f, 0.f)};                  // this thread's share of the rows' sums
        auto bias_of = [&](int k) { return m_ref[k] > -1e30f ? lvsc - m_ref[k] : lvsc; };
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const int s = j % NSC, base = tile_base(j), end = is_tail(j) ? c.total : c.n8;      // (a tile's tokens lie before `end`)
            ok = wait_bar(SC_FULL + s, j / NSC) && wait_bar(S_FULL + sbuf(q, j), sph(j));
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc_fence_after();
            const float* kn = reinterpret_cast<const float*>(smem + P::OFF_SC + s * P::SC) + t2;
            const float* vn = kn + TN;
            const uint32_t s_col = t_frag + sbuf(q, j) * TN;
            constexpr int NR = TN / 8;
            uint32_t v[4 * NR];                                    // of eight columns: two of row g, two of row g + 8
            tmem_ld_frag64(s_col, v);
            u64 nv[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) nv[r] = *reinterpret_cast<const u64*>(kn + 8 * r);
            tmem_ld_wait();
            // t = score * key scale - reference + log2(value scale)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t* x = v + 2 * k;
                const float bias = bias_of(k);
                const u64 b2 = pk(bias, bias);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float x0, x1;
                    upk(fma2(pk(__uint_as_float(x[4 * r]), __uint_as_float(x[4 * r + 1])), nv[r], b2), x0, x1);
                    x[4 * r] = __float_as_uint(x0); x[4 * r + 1] = __float_as_uint(x1);
                }
            }
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
            const uint2 spoilt = *reinterpret_cast<const uint2*>(smem + P::OFF_SC + s * P::SC + 2 * TN * 4);
            if (spoilt.x | spoilt.y) {                             // values that are not finite: NaN for the rows that see them
#pragma unroll
                for (int r = 0; r < 2 * NR; ++r) {
                    const int at = 8 * (r >> 1) + (r & 1) + t2;
                    if (((r < NR ? spoilt.x : spoilt.y) >> (at & 31)) & 1)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (v[4 * (r >> 1) + 2 * k + (r & 1)] != 0xff800000u) v[4 * (r >> 1) + 2 * k + (r & 1)] = 0x7fffffffu;
                }
            }
            // Weights, their sums, P = weight * value scale (both carry vsc) as fp16.  A row needs another reference when a weight exceeds
            // 2^MAX_SLACK, which its sum then does too: the sums are looked at behind the exponentials and no maximum is taken in the common case.
            // The lanes share the check of the tile's value scales, eight tokens' pairs each.
            const float2 v2 = *reinterpret_cast<const float2*>(vn + 8 * g);
            float vmax = fmaxf(v2.x, v2.y);
#pragma unroll
            for (int r = 0; r < NR; ++r) nv[r] = *reinterpret_cast<const u64*>(vn + 8 * r);
            uint32_t w[2 * NR];
            u64 ls[2];
#pragma unroll 1
            for (int pass = 0;; ++pass) {
                ls[0] = ls[1] = pk(0.f, 0.f);
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u64 x = pk(ex2(__uint_as_float(v[4 * r + 2 * k])), ex2(__uint_as_float(v[4 * r + 2 * k + 1])));
                        ls[k] = add2(ls[k], x);
                        float x0, x1;
                        upk(mul2(x, nv[r]), x0, x1);
                        w[2 * r + k] = pack_h2(x0, x1);
                    }
                bool again = vmax > vthr;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x0, x1;
                    upk(ls[k], x0, x1);
                    again = again || x0 + x1 > (m_ref[k] > -1e30f ? float(1 << int(MAX_SLACK)) * vsc : pos[k] >= base ? -1.f : INFINITY);      // (a row's first token: always)
                }
                if (pass > 0 || !__any_sync(0xffffffffu, again)) break;
                // Reference maximum / value scale: refreshed for the whole warp when any row needs it (rare after the first tile):
                // the rows' sums and their O in tensor memory are rescaled.
                float a[2], bias[2] = {bias_of(0), bias_of(1)}, mx[2] = {-INFINITY, -INFINITY}, ratio = 1.f;
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
                    const float nsc = __int_as_float((261 - eb) << 23);    // the largest value scale lands in [128, 256)
                    ratio = nsc / vsc;
                    vsc = nsc;
                    vthr = VSC_CAP / nsc;
                    lvsc = float(134 - eb);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float mn = fmaxf(fmaxf(m_ref[k], mx[k] - bias[k]), -1e30f);
                    a[k] = ex2(m_ref[k] - mn) * ratio;
                    m_ref[k] = mn;
                    const float delta = bias_of(k) - bias[k];
                    l2[k] = mul2(l2[k], pk(a[k], a[k]));
                    uint32_t* x = v + 2 * k;
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        x[4 * r] = __float_as_uint(__uint_as_float(x[4 * r]) + delta);
                        x[4 * r + 1] = __float_as_uint(__uint_as_float(x[4 * r + 1]) + delta);
                    }
                }
                if (j > 0) {
                    ok = wait_bar(O_DONE + q, j - 1);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < DP; c0 += 32) {
                        uint32_t o[16];
                        tmem_ld_frag32(t_frag + P::COL_O + q * DP + c0, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a[(i >> 1) & 1]);
                        tmem_st_frag32(t_frag + P::COL_O + q * DP + c0, o);
                    }
                    tmem_st_wait();
                }
            }
            if (!ok) break;
            l2[0] = add2(l2[0], ls[0]);
            l2[1] = add2(l2[1], ls[1]);
            tmem_st_half64(s_col, w);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar(P_FULL + sbuf(q, j)));
            mbar_arrive(bar(SC_FREE + s));
        }
        // ---- the rows' results, still as fragments: 32 bytes of a row from four lanes
        float l_sum[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float l1;
            upk(l2[k], l_sum[k], l1);
            l_sum[k] += l1;
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) l_sum[k] += __shfl_xor_sync(0xffffffffu, l_sum[k], off);
        }
        if (ok && n > 0) ok = wait_bar(ALL_DONE + q, 0);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const bool done = n > 0 && ok, parts = p.n_splits > 1;
        float* const part = parts ? p.part + (((int64_t(y) * p.n_blk + blk) * p.n_splits + split) * (NQ * TM) + mf) * (D + 4) : nullptr;
        if (parts && t2 == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) *reinterpret_cast<float2*>(part + k * 8 * (D + 4) + D) = done ? make_float2(m_ref[k] - lvsc, l_sum[k]) : make_float2(-INFINITY, 0.f);
        }
        if (done) {
            const bool f16 = c.dtype == TQ_F16, odd = (t2 & 2) != 0;
            float il[2];
            bool store[2];
            char* dst[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                il[k] = parts ? 1.f : 1.f / l_sum[k];
                store[k] = parts || row_valid(mf + 8 * k);
                dst[k] = parts ? reinterpret_cast<char*>(part + k * 8 * (D + 4) + t2) : static_cast<char*>(c.out) + 2 * (row_out(mf + 8 * k) + (t2 & 4) + (odd ? 8 : 0));
            }
            auto rows = [&](int c0, uint32_t (&o)[16]) {           // of eight columns: two of row g, two of row g + 8
                tmem_ld_frag32(t_frag + P::COL_O + q * DP + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * il[(i >> 1) & 1]);
            };
            if (parts) {
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[16];
                    rows(c0, o);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) *reinterpret_cast<uint2*>(dst[(i >> 1) & 1] + 4 * c0 + 8 * (i & 12)) = make_uint2(o[i], o[i + 1]);
                }
            } else {
                // two neighbouring lanes trade words: four columns each, the even one of eight columns, the odd one of the next eight
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[16];
                    rows(c0, o);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float x = __uint_as_float(o[i]), z = __uint_as_float(o[i + 1]);
                        o[i] = f16 ? pack_h2(x, z) : pack_bf2(x, z);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += (i & 2) ? 6 : 2) {
                        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? o[i] : o[i + 4], 1);
                        if (store[(i >> 1) & 1]) *reinterpret_cast<uint2*>(dst[(i >> 1) & 1] + 2 * c0 + 4 * (i & 12)) = odd ? make_uint2(other, o[i + 4]) : make_uint2(o[i], other);
                    }
                }
            }
        }
    } else {
        // ======================= softmax warps without a row: the others' exponentials have the pipe to themselves =======================
        // (What they leave in tensor memory meets rows that nobody reads.  A score buffer is full again only behind the products that every warp of
        // the query tile has arrived for, so that no arrival is a phase early.)
        const int q = warp >> 3;
        for (int j = 0; j < n; ++j) {
            if (!__all_sync(0xffffffffu, wait_bar(SC_FULL + j % NSC, j / NSC) && wait_bar(S_FULL + sbuf(q, j), sph(j)))) break;
            mbar_arrive(bar(P_FULL + sbuf(q, j)));
            mbar_arrive(bar(SC_FREE + j % NSC));
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

// A warp per query row: the ranges' partials in their order
template <int D> __global__ void __launch_bounds__(256) blocks_fa_merge_kernel(const __grid_constant__ Params p, int64_t n_rows) {
    constexpr int ROWS = Plan<D>::NQ * TM, NV = D / 32;
    const BlockAttendParams& c = p.a;
    const int lane = threadIdx.x & 31;
    const int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);               // row of the launch: (lane x head group, row block, row)
    pdl_wait();
    if (i >= n_rows) return;
    const int m = int(i % ROWS), blk = int(i / ROWS % p.n_blk), y = int(i / ROWS / p.n_blk);
    const int lane_c = y / p.HG, hg = y - lane_c * p.HG, b = lane_c / c.Hkv, hkv = lane_c - b * c.Hkv;
    const int tok = blk * Plan<D>::NQ * p.QT + (m >> 7) * p.QT + (m & 127) / p.GP, hh = (m & 127) % p.GP;
    if (hh >= min(HPG, c.G - hg * HPG) || tok >= c.Tq) return;
    const float* part = p.part + ((int64_t(y) * p.n_blk + blk) * p.n_splits * ROWS + m) * (D + 4);
    const int64_t stride = int64_t(ROWS) * (D + 4);
    float mm = -INFINITY, ll = 0.f;
    if (lane < p.n_splits) { mm = part[lane * stride + D]; ll = part[lane * stride + D + 1]; }
    float top = mm;
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float a = lane < p.n_splits && mm > -INFINITY ? ex2(mm - top) : 0.f;
    float sum = a > 0.f || ll != ll ? a * ll : 0.f;
#pragma unroll
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    float x[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = 0.f;
    for (int s = 0; s < p.n_splits; ++s) {
        const float w = __shfl_sync(0xffffffffu, a, s);
        const bool there = __shfl_sync(0xffffffffu, mm, s) > -INFINITY;            // (a range without a tile left no sums)
        if (!there) continue;
#pragma unroll
        for (int k = 0; k < NV; ++k) x[k] += w * part[s * stride + k * 32 + lane];
    }
    const int64_t out = ((int64_t(b) * c.Hq + hkv * c.G + hg * HPG + hh) * c.Tq + tok) * D + lane;
    const float il = 1.f / sum;
#pragma unroll
    for (int k = 0; k < NV; ++k) store_from_f32(c.out, c.dtype, out + k * 32, x[k] * il);
}

// Row blocks, and key ranges per row block: as many as shorten the whole launch, a CTA costing its tiles and some twelve more for set-up, first scores
// and the partials.
struct Shape { int HG, GP, QT, n_blk, n_splits; int64_t ctas; size_t part_bytes; };
template <int D> Shape shape_of(const BlockAttendParams& p) {
    Shape s{};
    const int g = std::min(p.G, HPG);
    s.HG = (p.G + HPG - 1) / HPG;
    s.GP = g <= 1 ? 1 : g <= 2 ? 2 : g <= 4 ? 4 : 8;
    s.QT = TM / s.GP;
    const int rows = Plan<D>::NQ * s.QT;
    s.n_blk = (p.Tq + rows - 1) / rows;
    const int64_t blocks = int64_t(p.B) * p.Hkv * s.HG * s.n_blk, sms = blocks_sm_count();
    const Visible v = visible_of(p.total, std::min(p.Tq, rows), p.window, p.sinks);            // of the last row block
    const int64_t tiles = (p.total - v.low + 63) / 64 + (v.sinks + 63) / 64 + 1;
    double best = 0.0;
    s.n_splits = 1;
    for (int n = 1; n <= MAX_RANGES && (n == 1 || tiles >= 2 * n); ++n) {
        const double t = double((blocks * n + sms - 1) / sms) * (double((tiles + n - 1) / n) + 12.0) + (n > 1 ? 8.0 : 0.0);
        if (n == 1 || t < best) { best = t; s.n_splits = n; }
    }
    s.ctas = blocks * s.n_splits;
    s.part_bytes = s.n_splits == 1 ? 0 : size_t(s.ctas) * Plan<D>::NQ * TM * (D + 4) * sizeof(float);
    return s;
}

template <int D> int launch(const BlockAttendParams& a, cudaStream_t st) {
    using P = Plan<D>;
    const Shape s = shape_of<D>(a);
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    if (dev < 0 || dev >= 64 || !set[dev].load()) {
        const cudaError_t e = cudaFuncSetAttribute(blocks_fa_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::SMEM));
        if (e != cudaSuccess) return fail(TQ_ERR_LAUNCH, "tq_blocks_attend: shared memory %zu B: %s", P::SMEM, cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) set[dev].store(true);
    }
    Params p{};
    p.a = a;
    p.HG = s.HG; p.GP = s.GP; p.QT = s.QT; p.n_blk = s.n_blk; p.n_splits = s.n_splits;
    p.part = a.part;
    if (!(p.status = decode_status_ptr())) return fail(TQ_ERR_LAUNCH, "tq_blocks_attend: cannot locate the status word");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(s.ctas));
    cfg.blockDim = dim3(P::NT);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, blocks_fa_kernel<D>, p);
    if (int rc = check_launch("tq_blocks_attend")) return rc;
    if (s.n_splits == 1) return TQ_OK;
    const int64_t rows = int64_t(s.ctas) / s.n_splits * P::NQ * TM;
    cfg.gridDim = dim3(unsigned((rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cudaLaunchKernelEx(&cfg, blocks_fa_merge_kernel<D>, p, rows);
    return check_launch("tq_blocks_attend");
}

}  // namespace bfa

// Whether this kernel takes the call: enough query rows per KV head for tiles of 128 to be worth their set-up
bool blocks_fa_takes(const BlockAttendParams& p) {
    if (p.dtype == TQ_F32 || (p.D != 64 && p.D != 96 && p.D != 128 && p.D != 256) || p.kn != nullptr) return false;
    return int64_t(p.Tq) * p.G >= 64 && int64_t(p.B) * p.Hkv * p.G * p.Tq < (int64_t(1) << 29);
}
size_t blocks_fa_workspace(const BlockAttendParams& p) {
    return p.D == 64 ? bfa::shape_of<64>(p).part_bytes : p.D == 96 ? bfa::shape_of<96>(p).part_bytes : p.D == 128 ? bfa::shape_of<128>(p).part_bytes : bfa::shape_of<256>(p).part_bytes;
}
int launch_blocks_fa(const BlockAttendParams& p, cudaStream_t s) {
    if (p.D == 64) return bfa::launch<64>(p, s);
    if (p.D == 96) return bfa::launch<96>(p, s);
    if (p.D == 128) return bfa::launch<128>(p, s);
    return bfa::launch<256>(p, s);
}

}  // namespace tq
