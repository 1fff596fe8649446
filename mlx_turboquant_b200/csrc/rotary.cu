// Rotary positions of queries and keys, from wherever a fused projection left them to the (B, H, L, D) rows that a cache takes, in one launch.
//
//   a' = m (a cos(p f) - b sin(p f)),  b' = m (b cos(p f) + a sin(p f))     for the pairs of the first `dims` coordinates; the rest is copied.
//
// Bound by memory: two bytes in and two out per coordinate.  A CTA owns a few tokens: it forms their cosines and sines once in shared memory,
// dims / 2 per token (angle and turns in float64, the fraction of a turn in float32), and all heads of the tokens use them.
// Measured: 8192 tokens x 40 heads of 128, bfloat16, 33 us = 5.0 TB/s (48 with one token at a time, 36 with 2.3 waves of CTAs); 4 tokens 5.8.
#include <algorithm>

#include "decode_dev.cuh"

namespace tq {

int blocks_sm_count();                                 // blocks.cu

namespace {

constexpr int RT = 256;                                // threads per CTA
constexpr int RT_ANGLES = 1024;                        // (cos, sin) pairs that a CTA has room for

struct RotaryParams {
    tq_rotary_rows part[2];
    int dtype, d, half, interleaved;                   // half: pairs per row
    int one_batch;
    int per_cta, groups;                               // tokens of a CTA; CTAs that share the heads of the same tokens
    int64_t tokens, length;                            // batch x length
    const double* freqs;
    float factor;
    int64_t offset;
    const int64_t* positions;
    int64_t pos_sb;
};

template <int VEC> struct Vec;                         // VEC 16-bit values
template <> struct Vec<8> { using T = uint4; };
template <> struct Vec<4> { using T = uint2; };
template <> struct Vec<2> { using T = uint32_t; };

template <typename E, int VEC> __device__ __forceinline__ void unpack(const typename Vec<VEC>::T& v, float (&x)[VEC]) {
    const E* e = reinterpret_cast<const E*>(&v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32<E>(e[i]);
}
template <typename E, int VEC> __device__ __forceinline__ typename Vec<VEC>::T pack(const float (&x)[VEC]) {
    typename Vec<VEC>::T v;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = sizeof(E) == 2 && std::is_same<E, __half>::value ? pack_h2(x[2 * i], x[2 * i + 1]) : pack_bf2(x[2 * i], x[2 * i + 1]);
    return v;
}

// cos and sin of position * freqs[i] times the factor.  In turns: the fraction of position * f / 2 pi is exact to 2^-53 of the turns, so that a
// position of 2^40 still has 13 bits of angle; sincospif's argument is in half turns.
__device__ __forceinline__ float2 turn_of(int64_t pos, double f, float factor) {
    const double turns = double(pos) * f * 0.15915494309189533577;
    float s, c;
    sincospif(float(2.0 * (turns - rint(turns))), &s, &c);
    return make_float2(c * factor, s * factor);
}

__device__ __forceinline__ void angles(const RotaryParams& p, float2* cs, int64_t tok0, int n_tok) {
    for (int i = threadIdx.x; i < n_tok * p.half; i += RT) {
        const int t = i / p.half, k = i - t * p.half;
        const int64_t tok = tok0 + t, b = tok / p.length, l = tok - b * p.length;
        cs[i] = turn_of(p.positions ? p.positions[b * p.pos_sb + l] : p.offset + l, p.freqs[k], p.factor);
    }
}

// 16-bit types, vectors of VEC coordinates: dims / 2 (half layout) or dims (interleaved), d, strides and addresses are multiples of VEC.
// A thread keeps one vector of the row (and its partner) and walks a run of the CTA's rows (token, head), ROWS loads under way at a time; the first ones are asked for
// before the angles are formed, and a token's cosines and sines stay in registers over its heads.
template <typename E, int VEC, bool INTERLEAVED> __global__ void __launch_bounds__(RT, 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
    using V = typename Vec<VEC>::T;
    constexpr int ROWS = 2, W = INTERLEAVED ? VEC / 2 : VEC;       // angles of a vector
    __shared__ __align__(16) float2 cs[RT_ANGLES];
    const int64_t grp = blockIdx.x / p.groups, tok0 = grp * p.per_cta;
    const int share = int(blockIdx.x - grp * p.groups), n_tok = int(min(int64_t(p.per_cta), p.tokens - tok0));
    const int heads = p.part[0].heads + p.part[1].heads;
    // vectors of a row: with their partners (half layout) or on their own (interleaved), then those that are copied
    const int turned = INTERLEAVED ? 2 * p.half / VEC : p.half / VEC, per_row = turned + (p.d - 2 * p.half) / VEC;
    const int h0 = heads * share / p.groups, nh = heads * (share + 1) / p.groups - h0, rows = n_tok * nh;
    const int sets = max(1, RT / per_row), set = threadIdx.x / per_row;
    const int run = (rows + sets - 1) / sets, r0 = set * run, r1 = set < sets ? min(r0 + run, rows) : 0;
    pdl_wait();
    pdl_trigger();
    auto walk = [&](int c, bool first_pass) {
        const bool copied = c >= turned;
        const int at = copied ? 2 * p.half + (c - turned) * VEC : c * VEC;
        int t = r0 / nh, h = h0 + r0 - t * nh, seen = -1;
        float2 w[W];
        V x[ROWS], y[ROWS];
        E* dst[ROWS];
        bool angles_there = !first_pass;
        for (int r = r0; r < r1 || !angles_there; r += ROWS) {
            int tt = t, hh = h, tok_of[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                if (r + u < r1) {
                    const int64_t tok = tok0 + tt, b = p.one_batch ? 0 : tok / p.length, l = tok - b * p.length;
                    const bool second = hh >= p.part[0].heads;
                    const tq_rotary_rows& q = p.part[second];
                    const int hq = second ? hh - p.part[0].heads : hh;
                    const E* src = static_cast<const E*>(q.x) + b * q.sb + hq * q.sh + l * q.st + at;
                    dst[u] = static_cast<E*>(q.out) + ((b * q.heads + hq) * p.length + l) * p.d + at;
                    x[u] = *reinterpret_cast<const V*>(src);
                    if (!INTERLEAVED && !copied) y[u] = *reinterpret_cast<const V*>(src + p.half);
                    tok_of[u] = tt;
                    if (++hh == h0 + nh) { hh = h0; ++tt; }
                }
            }
            t = tt; h = hh;
            if (!angles_there) {
                angles(p, cs, tok0, n_tok);
                __syncthreads();
                angles_there = true;
            }
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                if (r + u >= r1) continue;
                if (copied) {
                    *reinterpret_cast<V*>(dst[u]) = x[u];
                    continue;
                }
                if (tok_of[u] != seen) {
                    seen = tok_of[u];
#pragma unroll
                    for (int j = 0; j < W; ++j) w[j] = cs[seen * p.half + c * W + j];
                }
                float a[VEC];
                unpack<E, VEC>(x[u], a);
                if (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const float e = a[2 * j], z = a[2 * j + 1];
                        a[2 * j] = e * w[j].x - z * w[j].y;
                        a[2 * j + 1] = z * w[j].x + e * w[j].y;
                    }
                } else {
                    float z[VEC];
                    unpack<E, VEC>(y[u], z);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float e = a[j], f = z[j];
                        a[j] = e * w[j % W].x - f * w[j % W].y;
                        z[j] = f * w[j % W].x + e * w[j % W].y;
                    }
                    *reinterpret_cast<V*>(dst[u] + p.half) = pack<E, VEC>(z);
                }
                *reinterpret_cast<V*>(dst[u]) = pack<E, VEC>(a);
            }
        }
    };
    if (per_row <= RT) {
        walk(threadIdx.x - set * per_row, true);
    } else {
        // rows of more vectors than there are threads: one row at a time, a thread every 256th of its vectors
        walk(threadIdx.x, true);
        for (int c = threadIdx.x + RT; c < per_row; c += RT) walk(c, false);
    }
}

// any type, size and alignment: a pair (or a copied coordinate) per thread
__global__ void __launch_bounds__(RT) rotary_any_kernel(const __grid_constant__ RotaryParams p) {
    __shared__ float2 cs[RT_ANGLES];
    const int64_t grp = blockIdx.x / p.groups, tok0 = grp * p.per_cta;
    const int share = int(blockIdx.x - grp * p.groups), n_tok = int(min(int64_t(p.per_cta), p.tokens - tok0));
    pdl_wait();
    pdl_trigger();
    angles(p, cs, tok0, n_tok);
    __syncthreads();
    const int heads = p.part[0].heads + p.part[1].heads, per_row = p.d - p.half;
    const int h0 = heads * share / p.groups, h1 = heads * (share + 1) / p.groups, n = n_tok * (h1 - h0) * per_row;
    for (int i = threadIdx.x; i < n; i += RT) {
        const int row = i / per_row, c = i - row * per_row, t = row / (h1 - h0);
        int h = h0 + row - t * (h1 - h0);
        const int64_t tok = tok0 + t, b = tok / p.length, l = tok - b * p.length;
        const bool second = h >= p.part[0].heads;
        const tq_rotary_rows& q = p.part[second];
        if (second) h -= p.part[0].heads;
        const int64_t src = b * q.sb + h * q.sh + l * q.st, dst = ((b * q.heads + h) * p.length + l) * p.d;
        if (c >= p.half) {
            store_from_f32(q.out, p.dtype, dst + p.half + c, load_as_f32(q.x, p.dtype, src + p.half + c));
        } else {
            const int i0 = p.interleaved ? 2 * c : c, i1 = p.interleaved ? 2 * c + 1 : c + p.half;
            const float2 u = cs[t * p.half + c];
            const float a = load_as_f32(q.x, p.dtype, src + i0), z = load_as_f32(q.x, p.dtype, src + i1);
            store_from_f32(q.out, p.dtype, dst + i0, a * u.x - z * u.y);
            store_from_f32(q.out, p.dtype, dst + i1, z * u.x + a * u.y);
        }
    }
}

template <typename E> void launch_rotary(const cudaLaunchConfig_t& cfg, const RotaryParams& p, int vec) {
    if (p.interleaved) {
        if (vec == 8) cudaLaunchKernelEx(&cfg, rotary_kernel<E, 8, true>, p);
        else if (vec == 4) cudaLaunchKernelEx(&cfg, rotary_kernel<E, 4, true>, p);
        else cudaLaunchKernelEx(&cfg, rotary_kernel<E, 2, true>, p);
    } else {
        if (vec == 8) cudaLaunchKernelEx(&cfg, rotary_kernel<E, 8, false>, p);
        else if (vec == 4) cudaLaunchKernelEx(&cfg, rotary_kernel<E, 4, false>, p);
        else cudaLaunchKernelEx(&cfg, rotary_kernel<E, 2, false>, p);
    }
}

}  // namespace
}  // namespace tq

extern "C" int tq_rotary(const tq_rotary_args* a, void* stream) {
    using namespace tq;
    if (!a) return fail(TQ_ERR_INVALID, "tq_rotary: null args");
    if (!dtype_ok(a->dtype)) return fail(TQ_ERR_INVALID, "tq_rotary: bad dtype %d", a->dtype);
    if (a->batch < 0 || a->length < 0 || a->d <= 0 || a->dims <= 0 || a->dims % 2 || a->dims > a->d || a->dims > 2 * RT_ANGLES || a->part[0].heads < 0 || a->part[1].heads < 0)
        return fail(TQ_ERR_INVALID, "tq_rotary: batch %d, length %lld, d %d, dims %d (even, at most d and %d), heads %d and %d", a->batch, (long long)a->length, a->d, a->dims,
                    2 * RT_ANGLES, a->part[0].heads, a->part[1].heads);
    RotaryParams p{};
    p.tokens = int64_t(a->batch) * a->length;
    const int heads = a->part[0].heads + a->part[1].heads;
    if (p.tokens == 0 || heads == 0) return TQ_OK;
    if (!a->freqs) return fail(TQ_ERR_INVALID, "tq_rotary: no frequencies");
    p.dtype = a->dtype; p.d = a->d; p.half = a->dims / 2; p.interleaved = a->interleaved != 0; p.length = a->length;
    p.one_batch = a->batch == 1;
    p.freqs = a->freqs; p.factor = a->factor; p.offset = a->offset; p.positions = a->positions; p.pos_sb = a->pos_sb;
    int vec = a->dtype == TQ_F32 ? 1 : 8;
    for (int i = 0; i < 2; ++i) {
        const tq_rotary_rows& r = a->part[i];
        p.part[i] = r;
        if (r.heads == 0) continue;
        if (!r.x || !r.out) return fail(TQ_ERR_INVALID, "tq_rotary: null rows");
        while (vec > 1 && (!aligned(r.x, 2 * vec) || !aligned(r.out, 2 * vec) || r.sb % vec || r.sh % vec || r.st % vec)) vec /= 2;
    }
    while (vec > 1 && (a->d % vec || (a->interleaved ? a->dims : a->dims / 2) % vec)) vec /= 2;
    // Tokens per CTA: some eight vectors a thread, so that the angles cost little, and whole waves of four CTAs per SM (8192 tokens x 40 heads, d = 128: 34 us with
    // 2.3 waves); heads shared between CTAs where there are fewer tokens than that.
    const int items = heads * std::max(1, (a->d - (a->interleaved ? 0 : a->dims / 2)) / vec);
    const int64_t sms = blocks_sm_count(), slots = 4 * sms, most = std::max<int64_t>(1, std::min<int64_t>(10 * RT / items, RT_ANGLES / p.half)), waves = (p.tokens + slots * most - 1) / (slots * most);
    p.per_cta = int((p.tokens + slots * waves - 1) / (slots * waves));
    p.groups = p.per_cta > 1 ? 1 : int(std::max<int64_t>(1, std::min<int64_t>({(int64_t(items) + RT - 1) / RT, 2 * sms / p.tokens, heads})));
    const int64_t blocks = (p.tokens + p.per_cta - 1) / p.per_cta * p.groups;
    if (blocks >= (int64_t(1) << 31)) return fail(TQ_ERR_UNSUPPORTED, "tq_rotary: too many tokens");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(RT);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (vec == 1) cudaLaunchKernelEx(&cfg, rotary_any_kernel, p);
    else if (a->dtype == TQ_F16) launch_rotary<__half>(cfg, p, vec);
    else launch_rotary<__nv_bfloat16>(cfg, p, vec);
    return check_launch("tq_rotary");
}
