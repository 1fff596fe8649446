// Attention over the 8-bit block cache: one new token per sequence, and few query rows per KV head; sliding window and sinks.
//
//   out = sum_j softmax_j(scale q.k_j) v_j,   k_j = kc_j ks, v_j = vc_j vs with one ks, vs for each block of tokens, tokens of the tail as they are
//
// blocks_attend_kernel: bound by the codes' bytes.  Work is a flat sequence of tiles (16 tokens) of all (lane, group of 8 query rows); a CTA of eight warps
// takes an equal run of it, whatever lanes that touches, a warp every eighth tile of a lane.  Codes go through a ring of each warp's own in shared memory
// (cp.async, 16 bytes a lane).  mma.sync with the tokens as M (scores) and the coordinates as M (values): eight query rows share every code.  (The products
// are tiny, N = 8: tcgen05 would want 64 rows of operands staged in shared memory.)  Which coordinate a fragment's row or column stands for is free as long
// as queries and results agree.
//   scores, int8: integer products m16n8k32 on the codes as they are; the query in fixed point, 22 bits of its largest element, in digits of 7 bits; the sums are
//     exact.  (Two digits, 15 bits, lose the small coordinates of a query that has one 1000 times as large: scores then move by per cents.  A third costs 2% at most: 8 x
//     32,810 tokens 26.7 -> 27.2 us.  As fp16 operands the key codes cost 80 of 476 instructions per tile of 16 tokens at d = 128; the card runs this kernel at its power limit,
//     so that instructions count beside bytes.)
//   scores, e4m3: fp16 operands (codes are exact in them, and queries, bfloat16 ones under a power of two).  (mma.sync on e4m3 operands costs more than the
//     conversions here: 404 instructions per tile against 376.)
//   values: fp16, exact for both kinds of codes, times the softmax weights under their block's scale as two fp16 parts, 22 bits: one part's rounding is as large as an fp16
//     result's own, and a tenth of a bfloat16 one's.  The second part costs 0 to 5% (64 sequences x 16,384 tokens, 8 KV heads of 128, bfloat16: 375 to 385 us with and 368 to 385
//     without it in turn, at the card's power limit; a window of 4096 34.2 and 34.7).
// Where few (lane, group)s have few tiles each, a cluster of CTAs shares one and joins its sums over distributed shared memory: one launch.
// blocks_merge_kernel: joins the partials of a row that several CTAs worked on, in their order: results do not depend on which one came first.
// Measured, 4 heads on 1 at d = 128: int8, 8 lanes x 700 tokens 8.1 us (launch, one tile's chain of latencies, the cluster's joining), 8 x 32,810 27.4 (2.4 TB/s: 19 us of
// loop, then the merge's launch), e4m3, 128 lanes x a window of 4096 32 to 35 (4 TB/s); int8, 512 lanes x 16,380 390 to 450 as the card is cooled (4.8 to 5.5 TB/s of the 6.55 that
// a copy reaches; at its power limit, some 1.5 GHz).
// blocks_plain_kernel: a warp per token on CUDA cores, float32 throughout: float32 tokens, head dims without a layout above.
#include <algorithm>
#include <atomic>
#include <climits>

#include "blocks.cuh"

namespace tq {

namespace {

// ---------------------------------------------------------------------------------------------------- float32, any head_dim
constexpr int PL_W = 4;                                // warps of a CTA: one query row
__global__ void __launch_bounds__(PL_W * 32) blocks_plain_kernel(const __grid_constant__ BlockAttendParams p) {
    constexpr int NV = BLOCKS_MAX_D / 32;
    __shared__ float so[PL_W][BLOCKS_MAX_D], sm[PL_W], sl[PL_W];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ti = blockIdx.x % p.Tq, h = blockIdx.x / p.Tq % p.Hq, b = blockIdx.x / p.Tq / p.Hq, kv = h / p.G, nv = p.D / 32;
    const int64_t lane_c = int64_t(b) * p.Hkv + kv;
    pdl_wait();
    float q[NV], o[NV], m = -INFINITY, l = 0.f;
    for (int i = 0; i < nv; ++i) {
        q[i] = load_as_f32(p.q, p.dtype, b * p.q_sb + h * p.q_sh + ti * p.q_st + i * 32 + lane) * p.scale_log2;
        o[i] = 0.f;
    }
    const int pos = p.total - p.Tq + ti;
    const int low = max(0, pos - p.window + 1), sinks = min(p.sinks, low), n = sinks + pos + 1 - low;
    for (int i = warp; i < n; i += PL_W) {
        const int j = i < sinks ? i : low + i - sinks;
        const bool in8 = j < p.n8, fresh = p.kn != nullptr && j == p.total - 1;
        const int64_t code = (lane_c * p.cap + j) * p.D + lane, sc = lane_c * (p.cap >> p.shift) + (j >> p.shift), row = (lane_c * p.block + (j - p.n8)) * p.D + lane;
        float s = 0.f;
        for (int e = 0; e < nv; ++e) {
            const float k = in8 ? (p.e4m3 ? e4m3_to_f32(p.kc[code + e * 32]) : float(int8_t(p.kc[code + e * 32])))
                                : fresh ? load_as_f32(p.kn, p.dtype, b * p.kn_sb + kv * p.kn_sh + e * 32 + lane) : load_as_f32(p.kt, p.dtype, row + e * 32);
            s = fmaf(q[e], k, s);
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (in8) s *= p.ks[sc];
        const float mn = fmaxf(fmaxf(m, s), -1e30f), a = exp2f(m - mn), w = exp2f(s - mn), vs = in8 ? w * p.vs[sc] : w;
        m = mn;
        l = l * a + w;
        for (int e = 0; e < nv; ++e) {
            const float v = in8 ? (p.e4m3 ? e4m3_to_f32(p.vc[code + e * 32]) : float(int8_t(p.vc[code + e * 32])))
                                : fresh ? load_as_f32(p.vn, p.dtype, b * p.vn_sb + kv * p.vn_sh + e * 32 + lane) : load_as_f32(p.vt, p.dtype, row + e * 32);
            o[e] = fmaf(vs, v, o[e] * a);
        }
    }
    for (int e = 0; e < nv; ++e) so[warp][e * 32 + lane] = o[e];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    __syncthreads();
    float top = -1e30f, sum = 0.f;
    for (int w = 0; w < PL_W; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < PL_W; ++w) sum += sl[w] * exp2f(sm[w] - top);
    for (int i = threadIdx.x; i < p.D; i += PL_W * 32) {
        float x = 0.f;
        for (int w = 0; w < PL_W; ++w) x += so[w][i] * exp2f(sm[w] - top);
        store_from_f32(p.out, p.dtype, ((int64_t(b) * p.Hq + h) * p.Tq + ti) * p.D + i, x / sum);
        if (p.kn != nullptr && h % p.G == 0) {         // the appended row joins the tail (every reader takes it from where it came)
            const int64_t row = (lane_c * p.block + (p.total - 1 - p.n8)) * p.D + i;
            store_from_f32(p.kt_w, p.dtype, row, load_as_f32(p.kn, p.dtype, b * p.kn_sb + kv * p.kn_sh + i));
            store_from_f32(p.vt_w, p.dtype, row, load_as_f32(p.vn, p.dtype, b * p.vn_sb + kv * p.vn_sh + i));
        }
    }
}

// ---------------------------------------------------------------------------------------------------- 16-bit tokens
constexpr int AW = 8;                                  // warps of a CTA

// A tile is 16 tokens.  Each warp has a ring of ST tiles of codes in shared memory, row by row in 16-byte pieces; piece `c` of row `r` sits at place c ^ swizzle(r),
// which keeps the fragment reads below free of bank conflicts.
template <int D> struct AttendPlan {
    static constexpr int PER_SM = D == 256 ? 1 : 2;    // CTAs per SM
    static constexpr int ST = D == 64 ? 6 : D == 96 ? 4 : 3;
    static constexpr int CPR = D / 16;                 // 16-byte pieces of a row
    static constexpr uint32_t SIDE = 16 * D, STAGE = 2 * SIDE + 16;          // keys, values, their scales
    static constexpr int KW = D / 16, VW = D / 32;     // words of a lane per key row (two a tile) and value row (four)
    static constexpr int RS = D + 4;                   // floats of a partial row: sums, maximum, sum of weights
    static constexpr size_t RING = size_t(AW) * ST * STAGE, RED = size_t(AW) * HPG * RS * 4, OWN = size_t(HPG) * RS * 4, QB = size_t(5) * KW * 32 * 4, SMEM = (RING > RED + OWN ? RING : RED + OWN) + QB;
};

struct AttendGrid {
    int n_units, n_sink, n_win, low_unit, tail_unit;   // tiles of a (lane, group): sink tokens, window tokens in blocks, the tail's from tail_unit on
    int groups, slots;                                 // groups of 8 query rows per lane; partials of one
    int cluster;                                       // CTAs of a (lane, group) that join their sums over distributed shared memory; 0: runs of tiles
    int merge;                                         // the merge kernel follows
    uint32_t per, jobs;                                // tiles of a CTA's run; lanes x groups
    double us;                                         // what the call is expected to cost
};

// Which coordinates a lane's words are: a lane of t (keys) or g (values) holds 16-byte pieces of a row where the row has enough of them for all lanes, else parts of one.
//   keys, words of 4 codes:   d = 128 pieces 2 t, 2 t + 1;   256 pieces 4 t ... + 3;   64 piece t;   96 pieces t (0 ... 3), then half a piece of the last two
//   values:                   d = 128 piece g;   256 pieces 2 g, + 1;   64 half of piece g / 2;   96 half of piece g / 2 (0 ... 3), then a quarter of the last two
template <int D> __device__ __forceinline__ int key_dim(int w, int t) {
    if (D == 96) return w < 4 ? 16 * t + 4 * w : 64 + 8 * t + 4 * (w - 4);
    return (D / 4) * t + 4 * w;
}
template <int D> __device__ __forceinline__ int value_dim(int w, int g) {
    if (D == 96) return w < 2 ? 8 * g + 4 * w : 64 + 4 * g;
    return (D / 8) * g + 4 * w;
}
// Place of piece c of row r.  A read of 16 bytes is eight lanes at a time.  Keys: two rows (g, g + 1) x four pieces; values: four rows (2 t) x two pieces; with 8 or 16
// pieces a row, 128 or 256 bytes, a row's low bits over the piece's do for both.  d = 64: eight bytes a value lane, sixteen lanes at a time, four rows x two pieces.
template <int D> __device__ __forceinline__ uint32_t place(int r, int c) {
    if (D == 128) return uint32_t(r * 8 + (c ^ (r & 7)));
    if (D == 256) return uint32_t(r * 16 + (c ^ ((c >> 3) * 2) ^ (((r ^ (r >> 1)) & 1) + ((r >> 2) & 1) * 4)));
    if (D == 64 || c < 4) return uint32_t(r * 4 + (c ^ ((r >> 1) & 3)));
    return uint32_t(64 + r * 2 + (c - 4));             // (d = 96: two regions)
}
template <int BYTES> __device__ __forceinline__ void ld_ring(uint32_t at, uint32_t* w) {
    if constexpr (BYTES == 16) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}
template <int D> __device__ __forceinline__ void key_row(uint32_t side, int r, int t, uint32_t* w) {
    if constexpr (D == 96) {
        ld_ring<16>(side + place<D>(r, t) * 16, w);
        ld_ring<8>(side + place<D>(r, 4 + (t >> 1)) * 16 + (t & 1) * 8, w + 4);
    } else {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) ld_ring<16>(side + place<D>(r, (D / 64) * t + i) * 16, w + 4 * i);
    }
}
template <int D> __device__ __forceinline__ void value_row(uint32_t side, int r, int g, uint32_t* w) {
    if constexpr (D == 64) ld_ring<8>(side + place<D>(r, g >> 1) * 16 + (g & 1) * 8, w);
    else if constexpr (D == 96) {
        ld_ring<8>(side + place<D>(r, g >> 1) * 16 + (g & 1) * 8, w);
        ld_ring<4>(side + place<D>(r, 4 + (g >> 2)) * 16 + (g & 3) * 4, w + 2);
    } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) ld_ring<16>(side + place<D>(r, (D / 128) * g + i) * 16, w + 4 * i);
    }
}

// What a lane knows of the query columns 2 t and 2 t + 1 of its group
struct Cols {
    float scale[2];                                    // softmax scale * log2(e) over the query's power of two
    int pos[2];                                        // position; below every token where the column is empty
    int pos_min, pos_max;                              // of the group
};

// Scores of 16 tokens (rows g, g + 8) times their scales -> running softmax -> the weights as the value products' operand, as fp16 and what that
// leaves.  tok: token of row g.
template <int D>
__device__ __forceinline__ void weights(float (&s)[4], float kn0, float kn1, float vn0, float vn1, bool masked, int tok, const Cols& c, int window, int sinks, WarpAcc<D, 0>& st,
                                        uint32_t (&bp)[2], uint32_t (&rest)[2]) {
    s[0] *= kn0 * c.scale[0]; s[1] *= kn0 * c.scale[1];
    s[2] *= kn1 * c.scale[0]; s[3] *= kn1 * c.scale[1];
    bool hide[4] = {false, false, false, false};
    if (masked) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = tok + 8 * (i >> 1), pos = c.pos[i & 1];
            hide[i] = j > pos || (pos - j >= window && j >= sinks);
            if (hide[i]) s[i] = -INFINITY;
        }
        if (hide[0] && hide[1]) vn0 = 0.f;
        if (hide[2] && hide[3]) vn1 = 0.f;
    }
    const float mx0 = fmaxf(s[0], s[2]), mx1 = fmaxf(s[1], s[3]), vmax = fmaxf(vn0, vn1);
    if (__any_sync(0xffffffffu, mx0 > st.mt[0] || mx1 > st.mt[1] || vmax > st.vt)) softmax_refresh<D, 0>(mx0, mx1, vmax, st);
    const float p0 = ex2(s[0] - st.m[0]), p1 = ex2(s[1] - st.m[1]), p2 = ex2(s[2] - st.m[0]), p3 = ex2(s[3] - st.m[1]);
    st.l[0] += p0 + p2;
    st.l[1] += p1 + p3;
    const float w0 = vn0 * st.vsc, w1 = vn1 * st.vsc;
    float x[4] = {p0 * w0, p1 * w0, p2 * w1, p3 * w1};
    if (masked) {                                      // (a hidden token's scale may be a NaN)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (hide[i]) x[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        bp[i] = movm_t(*reinterpret_cast<const uint32_t*>(&h));
        const float2 hf = __half22float2(h);
        rest[i] = movm_t(pack_h2(x[2 * i] - hf.x, x[2 * i + 1] - hf.y));
    }
}

// Integer products, 16 tokens x 8 queries x 32 coordinates
__device__ __forceinline__ void mma_codes(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A query's four coordinates in N digits of 7 bits, the largest first: a word of four for each
template <int N> __device__ __forceinline__ void digits_of(const float (&x)[4], uint32_t (&w)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) w[n] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int r = __float2int_rn(x[i]);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int sh = 7 * (N - 1 - n), d = sh ? (r + (1 << (sh - 1))) >> sh : r;
            r -= d << sh;
            w[n] |= uint32_t(d & 255) << (8 * i);
        }
    }
}

// (128 registers at two CTAs an SM: the bfloat16 instances spill some 50 to 190 bytes, d = 64 none; the fp16 ones, whose loop over the blocks is the same and whose tail needs no conversion, none.)
template <int D, bool E4M3, bool BF> __global__ void __launch_bounds__(AW * 32, AttendPlan<D>::PER_SM) blocks_attend_kernel(const __grid_constant__ BlockAttendParams p, const __grid_constant__ AttendGrid z) {
    using P = AttendPlan<D>;
    constexpr int ST = P::ST, N = E4M3 ? 2 : 3;       // words of a query's four coordinates: fp16 pairs, or digits
    constexpr bool bf = BF;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    // a run of tiles, or the rank's share of a (lane, group)
    uint32_t u_first = blockIdx.x * z.per, u_last = min(u_first + z.per, z.jobs * uint32_t(z.n_units));
    if (z.cluster) {
        const uint32_t job = blockIdx.x / uint32_t(z.cluster), rank = blockIdx.x - job * uint32_t(z.cluster), n = uint32_t(z.n_units);
        u_first = job * n + n * rank / uint32_t(z.cluster);
        u_last = job * n + n * (rank + 1) / uint32_t(z.cluster);
    }
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + uint32_t(warp) * ST * P::STAGE;
    const int n_code = z.n_sink + z.n_win;
    bool waited = false;                               // (what only the parameters say is worked out before the kernel in front has ended)

    for (uint32_t at = u_first; at < u_last;) {
        const uint32_t job = at / uint32_t(z.n_units), lane_u = job / uint32_t(z.groups);
        const int u0 = int(at - job * uint32_t(z.n_units)), u1 = int(min(uint32_t(z.n_units), u0 + (u_last - at)));
        at += uint32_t(u1 - u0);
        const int grp = int(job - lane_u * uint32_t(z.groups)), b = int(lane_u / uint32_t(p.Hkv)), kv = int(lane_u) - b * p.Hkv;
        const int64_t lane_c = lane_u;

        // ---- queries and this warp's first tiles of codes are asked for
        const uint8_t* kc = p.kc + lane_c * p.cap * D + lane * 16;
        const uint8_t* vc = p.vc + lane_c * p.cap * D + lane * 16;
        const float* sc = (lane ? p.vs : p.ks) + lane_c * (p.cap >> p.shift);
        const int jump = (z.low_unit - z.n_sink) * 16;
        auto base_of = [&](int u) { return u * 16 + (u < z.n_sink ? 0 : jump); };
        const int end = min(u1, n_code);
        int next = u0 + warp;                          // the next tile to be asked for
        uint32_t fill = ring, use = ring;              // its place in the ring; the place of the tile at hand
        auto ask = [&]() {
            if (next < end) {
                const int base = base_of(next);
                const uint8_t* ks = kc + int64_t(base) * D;
                const uint8_t* vs = vc + int64_t(base) * D;
#pragma unroll
                for (int i = 0; i < (16 * P::CPR + 31) / 32; ++i) {
                    // (rows are 16 pieces or fewer: a lane's i-th piece is 32 / CPR rows further down)
                    const int x = lane + 32 * i, r = x / P::CPR;
                    const uint32_t dst = fill + place<D>(r, x - r * P::CPR) * 16;
                    cp_async16(dst, ks + 512 * i, 16);
                    cp_async16(dst + P::SIDE, vs + 512 * i, 16);
                }
                if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(fill + 2 * P::SIDE + 4 * lane), "l"(sc + (base >> p.shift)) : "memory");
            }
            cp_async_commit();
            next += AW;
            fill = fill == ring + (ST - 1) * P::STAGE ? ring : fill + P::STAGE;
        };
        const int rows = min(HPG, p.Tq * p.G - grp * HPG), r0 = grp * HPG;
        const char* q_row;                             // row g's
        {
            const int r = min(r0 + g, r0 + rows - 1), ti = r / p.G, h = kv * p.G + r - ti * p.G;
            q_row = static_cast<const char*>(p.q) + 2 * (b * p.q_sb + h * p.q_sh + ti * p.q_st);
        }
        if (!waited) {
            pdl_wait();
            pdl_trigger();
            waited = true;
        }
        uint2 qx[P::KW];
#pragma unroll
        for (int w = 0; w < P::KW; ++w) {
            qx[w] = *reinterpret_cast<const uint2*>(q_row + 2 * key_dim<D>(w, t));
            if (g >= rows) qx[w] = make_uint2(0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) ask();
        // ---- the group's queries as B operands (row g's coordinates in the order of the key codes)
        Cols c;
        uint32_t bq[N][P::KW];
        auto f4 = [&](uint2 v, float (&x)[4], float f) {
            if (bf) {
                x[0] = __uint_as_float(v.x << 16) * f; x[1] = __uint_as_float(v.x & 0xffff0000u) * f; x[2] = __uint_as_float(v.y << 16) * f; x[3] = __uint_as_float(v.y & 0xffff0000u) * f;
            } else {
                const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
                x[0] = lo.x * f; x[1] = lo.y * f; x[2] = hi.x * f; x[3] = hi.y * f;
            }
        };
        auto mag = [](uint2 v) { const uint32_t m = 0x7fff7fffu, y = __vmaxu2(v.x & m, v.y & m); return max(y & 0xffffu, y >> 16); };
        uint32_t* sq = reinterpret_cast<uint32_t*>(smem + P::SMEM - P::QB);
        float q_max;
        {
            // every warp looks at the whole query (its scale), and turns a word in eight of it into operands for all
            uint32_t mx = 0;
#pragma unroll
            for (int w = 0; w < P::KW; ++w) mx = max(mx, mag(qx[w]));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            q_max = bf ? __uint_as_float(mx << 16) : __half2float(__ushort_as_half(uint16_t(mx)));
            // e4m3: bfloat16 queries under the power of two that takes the largest element to [2^7, 2^8); int8: the largest element in N digits of 7 bits
            float f = E4M3 ? (bf ? stage_scale(__float_as_uint(q_max)) : 1.f) : q_max > 0.f ? fminf(2080000.f / q_max, 3.4028235e38f) : 1.f;
            if (!E4M3 && !(q_max <= 3.4028235e38f)) f = __uint_as_float(0x7fffffffu);       // (integers know no NaN: the scale is one)
#pragma unroll
            for (int w = 0; w < P::KW; ++w) {
                if ((w & (AW - 1)) != warp) continue;
                float y[4];
                uint32_t part[N];
                f4(qx[w], y, f);
                if constexpr (E4M3) {
                    part[0] = bf ? pack_h2(y[0], y[1]) : qx[w].x;
                    part[1] = bf ? pack_h2(y[2], y[3]) : qx[w].y;
                } else {
                    digits_of<N>(y, part);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) sq[(n * P::KW + w) * 32 + lane] = part[n];
                *reinterpret_cast<uint2*>(sq + ((3 * P::KW + 2 * w) * 32 + 2 * lane)) = qx[w];       // (for the tail)
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < P::KW; ++w)
#pragma unroll
                for (int n = 0; n < N; ++n) bq[n][w] = sq[(n * P::KW + w) * 32 + lane];
            const float inv = p.scale_log2 / f;
            const int first = p.total - p.Tq;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c.scale[i] = __shfl_sync(0xffffffffu, inv, 4 * (2 * t + i));
                c.pos[i] = 2 * t + i < rows ? first + (r0 + 2 * t + i) / p.G : -1;
            }
            c.pos_min = first + r0 / p.G;
            c.pos_max = first + (r0 + rows - 1) / p.G;
        }
        WarpAcc<D, 0> st;
        st.init();
        st.m[0] = st.m[1] = -1e30f;
        const int lo_min = c.pos_min - p.window + 1, lo_max = c.pos_max - p.window + 1;      // (the window's first token of the first and the last query)
        auto hidden = [&](int base) { return base > c.pos_max || (base + 15 < lo_min && base >= p.sinks); };
        auto whole = [&](int base) { return base + 15 <= c.pos_min && (base >= lo_max || base + 15 < p.sinks); };

        // ---- blocks
#pragma unroll 1
        for (int u = u0 + warp; u < end; u += AW) {
            cp_async_wait<ST - 2>();
            __syncwarp();
            ask();
            const uint32_t src = use;
            use = use == ring + (ST - 1) * P::STAGE ? ring : use + P::STAGE;
            const int tok = base_of(u);
            if (hidden(tok)) continue;
            uint32_t scales[2];
            ld_ring<8>(src + 2 * P::SIDE, scales);
            float s[4];
            {
                uint32_t k0[P::KW], k1[P::KW];
                key_row<D>(src, g, t, k0);
                key_row<D>(src, g + 8, t, k1);
                if constexpr (E4M3) {
                    float s2[4] = {0.f, 0.f, 0.f, 0.f};
                    s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
                    for (int w = 0; w < P::KW; ++w) {
                        uint32_t a[4];
                        halves<true>(k0[w], a[0], a[2]);
                        halves<true>(k1[w], a[1], a[3]);
                        mma16816((w & 1) ? s2 : s, a[0], a[1], a[2], a[3], bq[0][w], bq[1][w]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[k] += s2[k];
                } else {
                    int acc[N][4];
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
#pragma unroll
                        for (int w = 0; w < P::KW; w += 2) mma_codes(acc[n], k0[w], k1[w], k0[w + 1], k1[w + 1], bq[n][w], bq[n][w + 1]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[k] = float(acc[0][k]) * 16384.f + float(acc[1][k] * 128 + acc[N - 1][k]);
                }
            }
            const float kn = __uint_as_float(scales[0]), vn = __uint_as_float(scales[1]);
            uint32_t bp[2], rest[2];
            weights<D>(s, kn, kn, vn, vn, !whole(tok), tok + g, c, p.window, p.sinks, st, bp, rest);
            uint32_t v[4][P::VW];
#pragma unroll
            for (int r = 0; r < 4; ++r) value_row<D>(src + P::SIDE, 2 * t + (r & 1) + 8 * (r >> 1), g, v[r]);
            // two tokens' bytes side by side are the pairs of the transposed operand: coordinates w, w + 1 and w + 2, w + 3
#pragma unroll
            for (int w = 0; w < P::VW; ++w) {
                uint32_t a[4], e[4];
                halves<E4M3>(__byte_perm(v[0][w], v[1][w], 0x5140), a[0], a[1]);
                halves<E4M3>(__byte_perm(v[2][w], v[3][w], 0x5140), a[2], a[3]);
                halves<E4M3>(__byte_perm(v[0][w], v[1][w], 0x7362), e[0], e[1]);
                halves<E4M3>(__byte_perm(v[2][w], v[3][w], 0x7362), e[2], e[3]);
                mma16816(st.o[2 * w], a[0], a[1], a[2], a[3], bp[0], bp[1]);
                mma16816(st.o[2 * w + 1], e[0], e[1], e[2], e[3], bp[0], bp[1]);
                mma16816(st.o[2 * w], a[0], a[1], a[2], a[3], rest[0], rest[1]);
                mma16816(st.o[2 * w + 1], e[0], e[1], e[2], e[3], rest[0], rest[1]);
            }
        }
        cp_async_wait<0>();
        // ---- the tail: 16-bit rows, bfloat16 ones each under its power of two
        const int t0 = max(u0, n_code);
#pragma unroll 1
        for (int u = t0 + ((warp - (t0 - u0)) & (AW - 1)); u < u1; u += AW) {
            const int tok = p.n8 + (z.tail_unit + u - n_code) * 16;
            if (hidden(tok)) continue;
            // (a row that no query sees reads as zeros: what it holds must not reach the sums)
            auto row = [&](int j, bool keys, bool& in) -> const char* {
                in = j < p.total && (j >= lo_min || j < p.sinks);
                const int r = in ? j - p.n8 : 0;
                if (p.kn != nullptr && j == p.total - 1)
                    return keys ? static_cast<const char*>(p.kn) + 2 * (b * p.kn_sb + kv * p.kn_sh) : static_cast<const char*>(p.vn) + 2 * (b * p.vn_sb + kv * p.vn_sh);
                return static_cast<const char*>(keys ? p.kt : p.vt) + 2 * (lane_c * p.block + r) * D;
            };
            auto half4 = [&](uint2& v, float f) {
                v.x = pack_h2(__uint_as_float(v.x << 16) * f, __uint_as_float(v.x & 0xffff0000u) * f);
                v.y = pack_h2(__uint_as_float(v.y << 16) * f, __uint_as_float(v.y & 0xffff0000u) * f);
            };
            uint2 k[2][P::KW], v[4][P::VW];
            bool k_in[2], v_in[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const char* src = row(tok + g + 8 * r, true, k_in[r]);
#pragma unroll
                for (int w = 0; w < P::KW; ++w) k[r][w] = *reinterpret_cast<const uint2*>(src + 2 * key_dim<D>(w, t));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const char* src = row(tok + 2 * t + (r & 1) + 8 * (r >> 1), false, v_in[r]);
#pragma unroll
                for (int w = 0; w < P::VW; ++w) v[r][w] = *reinterpret_cast<const uint2*>(src + 2 * value_dim<D>(w, g));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int w = 0; w < P::KW; ++w)
                    if (!k_in[r]) k[r][w] = make_uint2(0u, 0u);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int w = 0; w < P::VW; ++w)
                    if (!v_in[r]) v[r][w] = make_uint2(0u, 0u);
            float kn[2] = {1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
            Cols ct = c;
            if (bf) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t mx = 0;
#pragma unroll
                    for (int w = 0; w < P::KW; ++w) mx = max(mx, mag(k[r][w]));
                    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float f = stage_scale(mx << 16);
                    kn[r] = 1.f / f;
#pragma unroll
                    for (int w = 0; w < P::KW; ++w) half4(k[r][w], f);
                }
            }
            {
                // the queries as fp16, bfloat16 ones under a power of two; c.scale is for the parts' scale
                const float qf = bf ? stage_scale(__float_as_uint(q_max)) : 1.f, inv = p.scale_log2 / qf;
#pragma unroll
                for (int w = 0; w < P::KW; ++w) {
                    uint2 x = *reinterpret_cast<const uint2*>(sq + ((3 * P::KW + 2 * w) * 32 + 2 * lane));
                    if (bf) half4(x, qf);
                    mma16816(s, k[0][w].x, k[1][w].x, k[0][w].y, k[1][w].y, x.x, x.y);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) ct.scale[i] = __shfl_sync(0xffffffffu, inv, 4 * (2 * t + i));
            }
            float f[4] = {1.f, 1.f, 1.f, 1.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t mx = 0;
#pragma unroll
                for (int w = 0; w < P::VW; ++w) mx = max(mx, mag(v[r][w]));
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                if (bf) {
                    f[r] = stage_scale(mx << 16);
#pragma unroll
                    for (int w = 0; w < P::VW; ++w) half4(v[r][w], f[r]);
                }
                // values that are not finite would reach queries that they are hidden from as 0 * inf: zeros, and a score of NaN
                if (mx >= (bf ? 0x7f80u : 0x7c00u)) {
                    f[r] = __uint_as_float(0x7fffffffu);
#pragma unroll
                    for (int w = 0; w < P::VW; ++w) v[r][w] = make_uint2(0u, 0u);
                }
            }
            float vn[2];                               // tokens g and g + 8 sit with the lane of t = g / 2
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float a = __shfl_sync(0xffffffffu, f[2 * r], g >> 1), e = __shfl_sync(0xffffffffu, f[2 * r + 1], g >> 1);
                vn[r] = 1.f / ((g & 1) ? e : a);
                if (vn[r] != vn[r]) { kn[r] = vn[r]; vn[r] = 0.f; }
            }
            uint32_t bp[2], rest[2];
            weights<D>(s, kn[0], kn[1], vn[0], vn[1], true, tok + g, ct, p.window, p.sinks, st, bp, rest);
#pragma unroll
            for (int w = 0; w < P::VW; ++w) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t x0 = i ? v[0][w].y : v[0][w].x, x1 = i ? v[1][w].y : v[1][w].x, x2 = i ? v[2][w].y : v[2][w].x, x3 = i ? v[3][w].y : v[3][w].x;
                    const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632), a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
                    mma16816(st.o[2 * w + i], a0, a1, a2, a3, bp[0], bp[1]);
                    mma16816(st.o[2 * w + i], a0, a1, a2, a3, rest[0], rest[1]);
                }
            }
        }
        if (p.kn != nullptr && grp == 0 && u1 == z.n_units) {          // whoever has the lane's last tile stores the appended row
            for (int i = tid; i < D / 4; i += AW * 32) {
                const int side = i >= D / 8, ch = (i - side * (D / 8)) * 8;
                const char* src = side ? static_cast<const char*>(p.vn) + 2 * (b * p.vn_sb + kv * p.vn_sh) : static_cast<const char*>(p.kn) + 2 * (b * p.kn_sb + kv * p.kn_sh);
                char* dst = static_cast<char*>(side ? p.vt_w : p.kt_w) + 2 * (lane_c * p.block + (p.total - 1 - p.n8)) * D;
                *reinterpret_cast<uint4*>(dst + 2 * ch) = *reinterpret_cast<const uint4*>(src + 2 * ch);
            }
        }
        // ---- the warps' sums into one, where the rings were
        __syncthreads();
        float* red = reinterpret_cast<float*>(smem);
        st.finish();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], off);
            float* row = red + (warp * HPG + 2 * t + i) * P::RS;
#pragma unroll
            for (int w = 0; w < P::VW; ++w)
                *reinterpret_cast<float4*>(row + value_dim<D>(w, g)) = make_float4(st.o[2 * w][i], st.o[2 * w][2 + i], st.o[2 * w + 1][i], st.o[2 * w + 1][2 + i]);
            if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(st.m[i], st.l[i]);
        }
        __syncthreads();
        const bool alone = u0 == 0 && u1 == z.n_units;
        const uint32_t slot = blockIdx.x - job * uint32_t(z.n_units) / z.per;
        auto store = [&](int r, int d0, const float (&x)[4], float l) {
            const int rr = r0 + r, ti = rr / p.G, h = kv * p.G + rr - ti * p.G;
            const float il = 1.f / l;
            char* dst = static_cast<char*>(p.out) + 2 * (((int64_t(b) * p.Hq + h) * p.Tq + ti) * D + d0);
            *reinterpret_cast<uint2*>(dst) = bf ? make_uint2(pack_bf2(x[0] * il, x[1] * il), pack_bf2(x[2] * il, x[3] * il)) : make_uint2(pack_h2(x[0] * il, x[1] * il), pack_h2(x[2] * il, x[3] * il));
        };
        float* own = red + AW * HPG * P::RS;           // (cluster)
        for (int i = tid; i < rows * (D / 4); i += AW * 32) {
            const int r = i / (D / 4), d0 = (i - r * (D / 4)) * 4;
            const float* row = red + r * P::RS;
            float top = -1e30f, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < AW; ++w) top = fmaxf(top, row[w * HPG * P::RS + D]);
#pragma unroll
            for (int w = 0; w < AW; ++w) {
                const float2 ml = *reinterpret_cast<const float2*>(row + w * HPG * P::RS + D);
                const float a = ex2(ml.x - top);
                const float4 v = *reinterpret_cast<const float4*>(row + w * HPG * P::RS + d0);
                l += a * ml.y;
                x[0] += a * v.x; x[1] += a * v.y; x[2] += a * v.z; x[3] += a * v.w;
            }
            if (alone) {
                store(r, d0, x, l);
            } else {
                float* part = z.cluster ? own + r * P::RS : p.part + ((int64_t(job) * z.slots + slot) * HPG + r) * P::RS;
                *reinterpret_cast<float4*>(part + d0) = make_float4(x[0], x[1], x[2], x[3]);
                if (d0 == 0) *reinterpret_cast<float2*>(part + D) = make_float2(top, l);
            }
        }
        if (z.cluster > 1) {
            // the ranks' sums, each rank its share of the group's coordinates, in the ranks' order
            const uint32_t rank = blockIdx.x % uint32_t(z.cluster), here = static_cast<uint32_t>(__cvta_generic_to_shared(own));
            asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
            for (int i = tid + int(rank) * AW * 32; i < rows * (D / 4); i += z.cluster * AW * 32) {
                const int r = i / (D / 4), d0 = (i - r * (D / 4)) * 4;
                float4 v[8];
                float2 ml[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    ml[k] = make_float2(-1e30f, 0.f);
                    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (k >= z.cluster) continue;
                    uint32_t at;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(here + uint32_t(r * P::RS * 4)), "r"(k));
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w) : "r"(at + 4 * d0) : "memory");
                    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(ml[k].x), "=f"(ml[k].y) : "r"(at + 4 * D) : "memory");
                }
                float top = -1e30f, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float a = ex2(ml[k].x - top);
                    l += a * ml[k].y;
                    x[0] += a * v[k].x; x[1] += a * v[k].y; x[2] += a * v[k].z; x[3] += a * v[k].w;
                }
                store(r, d0, x, l);
            }
            asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // (a rank's memory stays until all have read it)
        }
        __syncthreads();
    }
}

// A CTA per query row that more than one CTA worked on: a thread has four coordinates and every n-th partial, so that all loads are under way at once
constexpr int MG_T = 128;
template <int D> __global__ void __launch_bounds__(MG_T) blocks_merge_kernel(const __grid_constant__ BlockAttendParams p, const __grid_constant__ AttendGrid z) {
    using P = AttendPlan<D>;
    constexpr int Q = D / 4, N = MG_T / Q;             // threads of a partial row; partials at a time
    __shared__ float4 sx[N][Q];
    __shared__ float2 sm[N];
    const uint32_t job = blockIdx.x / HPG, lane_u = job / uint32_t(z.groups);
    const int r = blockIdx.x % HPG, grp = int(job - lane_u * uint32_t(z.groups)), rr = grp * HPG + r;
    const int set = threadIdx.x / Q, d0 = threadIdx.x - set * Q;
    if (rr >= p.Tq * p.G) return;
    const uint32_t c0 = job * uint32_t(z.n_units) / z.per, c1 = ((job + 1) * uint32_t(z.n_units) - 1) / z.per;
    if (c0 == c1) return;
    const int n = int(c1 - c0) + 1;
    const float* part = p.part + (int64_t(job) * z.slots * HPG + r) * P::RS;
    constexpr int STEP = HPG * P::RS;
    pdl_wait();
    pdl_trigger();
    float m = -1e30f, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (set < N) {
        for (int s = set; s < n; s += 8 * N) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float* q = part + int64_t(s + i * N < n ? s + i * N : s) * STEP;
                ml[i] = *reinterpret_cast<const float2*>(q + D);
                v[i] = *reinterpret_cast<const float4*>(q + 4 * d0);
                if (s + i * N >= n) { ml[i] = make_float2(-1e30f, 0.f); v[i] = make_float4(0.f, 0.f, 0.f, 0.f); }
            }
            float top = m;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, ml[i].x);
            const float a0 = ex2(m - top);
            l *= a0; x.x *= a0; x.y *= a0; x.z *= a0; x.w *= a0;
            m = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = ex2(ml[i].x - top);
                l += a * ml[i].y;
                x.x += a * v[i].x; x.y += a * v[i].y; x.z += a * v[i].z; x.w += a * v[i].w;
            }
        }
        sx[set][d0] = x;
        if (d0 == 0) sm[set] = make_float2(m, l);
    }
    __syncthreads();
    if (threadIdx.x >= Q) return;
    float top = -1e30f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, sm[i].x);
    l = 0.f;
    x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float a = ex2(sm[i].x - top);
        const float4 v = sx[i][d0];
        l += a * sm[i].y;
        x.x += a * v.x; x.y += a * v.y; x.z += a * v.z; x.w += a * v.w;
    }
    const int b = int(lane_u / uint32_t(p.Hkv)), kv = int(lane_u) - b * p.Hkv, ti = rr / p.G, h = kv * p.G + rr - ti * p.G;
    const float il = 1.f / l;
    char* dst = static_cast<char*>(p.out) + 2 * (((int64_t(b) * p.Hq + h) * p.Tq + ti) * D + 4 * d0);
    *reinterpret_cast<uint2*>(dst) = p.dtype == TQ_BF16 ? make_uint2(pack_bf2(x.x * il, x.y * il), pack_bf2(x.z * il, x.w * il)) : make_uint2(pack_h2(x.x * il, x.y * il), pack_h2(x.z * il, x.w * il));
}

// How many clusters of each size the card holds at a time (a cluster lies within one group of SMs, so 148 SMs hold fewer of
// six or seven CTAs than their number says).
template <int D> int clusters_at_once(int size) {
    using P = AttendPlan<D>;
    static std::atomic<int> known[64][9];                  // (zero: not asked yet)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 0; }
    int n = known[dev][size].load();
    if (n != 0) return n;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(size) * 512);
    cfg.blockDim = dim3(AW * 32);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(blocks_attend_kernel<D, false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::SMEM)) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, blocks_attend_kernel<D, false, false>, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = blocks_sm_count() * P::PER_SM / size;
    }
    known[dev][size].store(n);
    return n;
}

template <int D> AttendGrid grid_of(const BlockAttendParams& p) {
    using P = AttendPlan<D>;
    const Visible v = visible_of(p.total, p.Tq, p.window, p.sinks);
    AttendGrid z{};
    const int code_units = p.n8 / 16;
    z.low_unit = std::min(v.low, p.n8) / 16;
    z.n_win = v.low >= p.n8 ? 0 : code_units - z.low_unit;
    z.n_sink = (std::min(v.sinks, p.n8) + 15) / 16;
    if (z.n_win > 0) z.n_sink = std::min(z.n_sink, z.low_unit);
    z.tail_unit = v.sinks > p.n8 ? 0 : std::max(v.low - p.n8, 0) / 16;
    z.n_units = z.n_sink + z.n_win + (p.total - p.n8 + 15) / 16 - z.tail_unit;
    z.groups = int((int64_t(p.Tq) * p.G + HPG - 1) / HPG);
    const int64_t jobs = int64_t(p.B) * p.Hkv * z.groups, units = jobs * z.n_units, ctas = int64_t(blocks_sm_count()) * P::PER_SM;
    if (units >= (int64_t(1) << 31) || jobs >= (int64_t(1) << 28)) { z.jobs = 0; z.us = 1e30; return z; }
    z.jobs = uint32_t(jobs);
    z.per = uint32_t(std::max<int64_t>(AW, (units + ctas - 1) / ctas));
    z.slots = std::min((z.n_units - 2) / int(z.per) + 2, z.n_units);
    z.merge = z.per % uint32_t(z.n_units) != 0;            // (otherwise every row has one CTA)
    const bool fits = !z.merge || size_t(jobs) * z.slots * HPG * P::RS * sizeof(float) <= p.room;
    // A (lane, group) in one launch, by a cluster of up to eight CTAs, or runs of tiles over the whole card and a merge.  In us, fitted to 190 calls at d = 64, 128 and 256
    // (8 to 256 lanes, 1 to 16 groups, 100 to 16,000 tokens; the choice is within 1% of the best on the mean, 20% at the worst): a tile at d = 128 0.15 with one CTA on an SM
    // and 0.18 with two, a wave of CTAs 7, every further (lane, group) in a run 12, a cluster's joining 2.5, the merge 8 and 4 for every thousand partials.
    const double width = D <= 64 ? 0.52 : D <= 96 ? 0.76 : D <= 128 ? 1.0 : 1.3;
    auto tile_us = [&](int64_t n) { return width * (P::PER_SM == 2 && n * 2 > ctas ? 0.18 : 0.15); };
    z.us = !fits ? 1e29 : double(z.per) * tile_us((units + z.per - 1) / z.per) + 7.0 + 12.0 * std::max(0.0, double(z.per) / z.n_units - 0.5) + (z.merge ? 8.0 + 0.004 * double(jobs) * z.slots : 0.0);
    for (int c = 1; c <= 8 && (c == 1 || c * AW <= z.n_units + AW - 1); ++c) {
        const int64_t n = c == 1 ? ctas : clusters_at_once<D>(c);
        if (n <= 0) continue;
        const double us = double((jobs + n - 1) / n) * (double((z.n_units + c - 1) / c) * tile_us(jobs * c) + 7.0) + (c > 1 ? 2.5 : 0.0);
        if (us < z.us) { z.us = us; z.cluster = c; z.merge = 0; }
    }
    return z;
}
template <int D> size_t split_workspace(const BlockAttendParams& p) {
    const AttendGrid z = grid_of<D>(p);
    if (!z.merge) return 0;
    return size_t(z.jobs) * z.slots * HPG * AttendPlan<D>::RS * sizeof(float);
}

template <int D> int split_choice(const BlockAttendParams& p) {
    const AttendGrid z = grid_of<D>(p);
    return z.cluster > 1 ? TQ_BLOCKS_CLUSTER : z.merge ? TQ_BLOCKS_RUNS : TQ_BLOCKS_ALONE;
}

template <int D> int launch_split(const BlockAttendParams& p, cudaStream_t s) {
    using P = AttendPlan<D>;
    const AttendGrid z = grid_of<D>(p);
    if (z.jobs == 0) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_attend: too many query rows");
    static std::atomic<bool> set[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    if (dev < 0 || dev >= 64 || !set[dev].load()) {
        cudaError_t e = cudaSuccess;
        for (auto* k : {blocks_attend_kernel<D, true, true>, blocks_attend_kernel<D, true, false>, blocks_attend_kernel<D, false, true>, blocks_attend_kernel<D, false, false>})
            if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::SMEM));
        if (e != cudaSuccess) return fail(TQ_ERR_LAUNCH, "tq_blocks_attend: shared memory %zu B: %s", P::SMEM, cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) set[dev].store(true);
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(std::max(z.cluster, 1));
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(z.cluster ? z.jobs * uint32_t(z.cluster) : (z.jobs * uint32_t(z.n_units) + z.per - 1) / z.per);
    cfg.blockDim = dim3(AW * 32);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = z.cluster > 1 ? 2 : 1;
    const bool bf = p.dtype == TQ_BF16;
    cudaLaunchKernelEx(&cfg, p.e4m3 ? (bf ? blocks_attend_kernel<D, true, true> : blocks_attend_kernel<D, true, false>)
                                    : (bf ? blocks_attend_kernel<D, false, true> : blocks_attend_kernel<D, false, false>), p, z);
    if (int rc = check_launch("tq_blocks_attend")) return rc;
    if (!z.merge) return TQ_OK;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(z.jobs * HPG);
    cfg.blockDim = dim3(MG_T);
    cfg.dynamicSmemBytes = 0;
    cudaLaunchKernelEx(&cfg, blocks_merge_kernel<D>, p, z);
    return check_launch("tq_blocks_attend");
}

bool split_takes(const BlockAttendParams& p) { return p.dtype != TQ_F32 && (p.D == 64 || p.D == 96 || p.D == 128 || p.D == 256); }

// Arguments -> parameters; done: nothing to compute
int prepare(const tq_blocks_attend_args* a, BlockAttendParams& p, bool& done) {
    const char* what = "tq_blocks_attend";
    if (!a) return fail(TQ_ERR_INVALID, "%s: null args", what);
    const tq_block_store& s = a->store;
    if (int rc = check_store(&s, what)) return rc;
    const bool append = a->k_new.x != nullptr;
    const int64_t total = s.length + (append ? 1 : 0);
    if (a->n_q_heads < 0 || a->t_q < 0 || (s.n_kv_heads > 0 && a->n_q_heads % s.n_kv_heads)) return fail(TQ_ERR_INVALID, "%s: %d query heads on %d", what, a->n_q_heads, s.n_kv_heads);
    if (a->window < 0 || a->sinks < 0) return fail(TQ_ERR_INVALID, "%s: window %lld, sinks %lld", what, (long long)a->window, (long long)a->sinks);
    if (append != (a->v_new.x != nullptr)) return fail(TQ_ERR_INVALID, "%s: new keys without values", what);
    if (append && (a->t_q != 1 || s.length % s.block + 1 >= s.block))
        return fail(TQ_ERR_INVALID, "%s: one new token that does not complete a block can be appended (%lld query tokens, length %lld)", what, (long long)a->t_q, (long long)s.length);
    if (a->t_q > total) return fail(TQ_ERR_INVALID, "%s: %lld query tokens over %lld in the cache", what, (long long)a->t_q, (long long)total);
    done = s.batch == 0 || a->n_q_heads == 0 || a->t_q == 0;
    if (done) return TQ_OK;
    if (s.n_kv_heads == 0 || !a->q.x || !a->out) return fail(TQ_ERR_INVALID, "%s: null queries or result", what);
    const int es = s.dtype == TQ_F32 ? 4 : 2;
    auto rows_ok = [&](const tq_new_rows& r, bool tokens) { return aligned(r.x, 16) && (r.sb * es) % 16 == 0 && (r.sh * es) % 16 == 0 && (!tokens || (r.st * es) % 16 == 0); };
    if (!rows_ok(a->q, true) || !aligned(a->out, 16) || (append && (!rows_ok(a->k_new, false) || !rows_ok(a->v_new, false))))
        return fail(TQ_ERR_UNSUPPORTED, "%s: rows must be 16-byte aligned", what);
    p = BlockAttendParams{};
    p.kc = static_cast<const uint8_t*>(s.k_codes); p.vc = static_cast<const uint8_t*>(s.v_codes); p.ks = s.k_scales; p.vs = s.v_scales;
    p.kt = p.kt_w = s.k_tail; p.vt = p.vt_w = s.v_tail;
    if (append) {
        p.kn = a->k_new.x; p.vn = a->v_new.x; p.kn_sb = a->k_new.sb; p.kn_sh = a->k_new.sh; p.vn_sb = a->v_new.sb; p.vn_sh = a->v_new.sh;
    }
    p.q = a->q.x; p.q_sb = a->q.sb; p.q_sh = a->q.sh; p.q_st = a->q.st;
    p.out = a->out; p.dtype = s.dtype; p.e4m3 = s.code_type == TQ_CODE_E4M3;
    p.B = s.batch; p.Hq = a->n_q_heads; p.Hkv = s.n_kv_heads; p.G = a->n_q_heads / s.n_kv_heads; p.D = s.d; p.Tq = int(a->t_q);
    p.block = s.block; p.shift = log2_of(s.block); p.cap = s.capacity;
    p.n8 = int(s.length / s.block * s.block); p.total = int(total);
    p.window = a->window > 0 ? int(std::min<int64_t>(a->window, INT_MAX / 2)) : INT_MAX / 2;
    p.sinks = int(std::min<int64_t>(a->sinks, INT_MAX / 2));
    p.scale_log2 = a->scale * LOG2E;
    if (a->workspace && !aligned(a->workspace, 256)) return fail(TQ_ERR_INVALID, "%s: the workspace must be 256-byte aligned", what);
    p.part = static_cast<float*>(a->workspace);
    p.room = a->workspace_bytes;
    return TQ_OK;
}

size_t workspace_of(const BlockAttendParams& p) {
    if (!split_takes(p)) return 0;
    if (blocks_fa_takes(p)) return blocks_fa_workspace(p);
    return p.D == 64 ? split_workspace<64>(p) : p.D == 96 ? split_workspace<96>(p) : p.D == 128 ? split_workspace<128>(p) : split_workspace<256>(p);
}

}  // namespace

double blocks_split_us(const BlockAttendParams& p) { return p.D == 64 ? grid_of<64>(p).us : p.D == 96 ? grid_of<96>(p).us : p.D == 128 ? grid_of<128>(p).us : grid_of<256>(p).us; }

int launch_blocks_plain(const BlockAttendParams& p, cudaStream_t s) {
    const int64_t rows = int64_t(p.B) * p.Hq * p.Tq;
    if (rows >= (int64_t(1) << 31)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_attend: too many query rows");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(rows));
    cfg.blockDim = dim3(PL_W * 32);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, blocks_plain_kernel, p);
    return check_launch("tq_blocks_attend");
}

}  // namespace tq

extern "C" size_t tq_blocks_attend_workspace_within(const tq_blocks_attend_args* a, size_t room) {
    tq::BlockAttendParams p;
    bool done = false;
    if (tq::prepare(a, p, done) != TQ_OK || done) return 0;
    p.room = room;
    return tq::workspace_of(p);
}

extern "C" size_t tq_blocks_attend_workspace(const tq_blocks_attend_args* a) { return tq_blocks_attend_workspace_within(a, SIZE_MAX); }

extern "C" int tq_blocks_attend_choice(const tq_blocks_attend_args* a) {
    tq::BlockAttendParams p;
    bool done = false;
    if (int rc = tq::prepare(a, p, done)) return rc;
    if (done) return TQ_BLOCKS_NOTHING;
    if (!tq::split_takes(p)) return TQ_BLOCKS_PLAIN;
    if (tq::blocks_fa_takes(p)) return tq::blocks_fa_choice(p);
    return p.D == 64 ? tq::split_choice<64>(p) : p.D == 96 ? tq::split_choice<96>(p) : p.D == 128 ? tq::split_choice<128>(p) : tq::split_choice<256>(p);
}

extern "C" int tq_blocks_attend(const tq_blocks_attend_args* a, void* stream) {
    using namespace tq;
    BlockAttendParams p;
    bool done = false;
    if (int rc = prepare(a, p, done)) return rc;
    if (done) return TQ_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!a->workspace) p.room = 0;
    if (!split_takes(p)) return launch_blocks_plain(p, s);
    if (blocks_fa_takes(p)) return launch_blocks_fa(p, s);
    if (p.D == 64) return launch_split<64>(p, s);
    if (p.D == 96) return launch_split<96>(p, s);
    if (p.D == 128) return launch_split<128>(p, s);
    return launch_split<256>(p, s);
}
