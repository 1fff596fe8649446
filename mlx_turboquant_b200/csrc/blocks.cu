// A cache held in 8 bits: tokens quantised as they are written, a scale for each block of tokens and head, and read back dense.
//
//   A = max |x| over the block's tokens x D;   int8: c = rint(x * (127 / A)), s = A / 127;   e4m3: c = e4m3(x * (448 / A)), s = A / 448
//
// in float32 with IEEE divisions.  A block is quantised once, when its last token arrives, so that the storage depends on the tokens alone and not on
// the calls they came in; the tokens behind the last whole block stay in a tail as they are.
//
// Both kernels are bound by memory.  Writing holds a block in registers between its maximum and its codes: one read of two bytes, one write of one
// byte a value.  Reading back moves one byte in and two (four) out (8 x 65,519 tokens, d = 128, both sides 402 MB: 64 us = 6.3 TB/s).
#include <algorithm>
#include <atomic>
#include <climits>

#include "blocks.cuh"

namespace tq {

int check_store(const tq_block_store* s, const char* what) {
    if (!s) return fail(TQ_ERR_INVALID, "%s: null store", what);
    if (!dtype_ok(s->dtype)) return fail(TQ_ERR_INVALID, "%s: bad dtype %d", what, s->dtype);
    if (s->code_type != TQ_CODE_INT8 && s->code_type != TQ_CODE_E4M3) return fail(TQ_ERR_INVALID, "%s: bad code type %d", what, s->code_type);
    if (!block_ok(s->block)) return fail(TQ_ERR_INVALID, "%s: blocks of %d tokens (16, 32, 64 or 128)", what, s->block);
    if (s->batch < 0 || s->n_kv_heads < 0 || s->capacity < 0 || s->capacity % s->block || s->length < 0)
        return fail(TQ_ERR_INVALID, "%s: batch %d, heads %d, capacity %lld (a multiple of the block), length %lld", what, s->batch, s->n_kv_heads, (long long)s->capacity,
                    (long long)s->length);
    if (s->length / s->block * s->block > s->capacity) return fail(TQ_ERR_INVALID, "%s: %lld tokens in storage for %lld", what, (long long)s->length, (long long)s->capacity);
    if (s->d <= 0 || s->d % 32 || s->d > BLOCKS_MAX_D) return fail(TQ_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 32 up to %d", what, s->d, BLOCKS_MAX_D);
    if (int64_t(s->batch) * s->n_kv_heads >= (1 << 24) || s->length >= (1 << 30)) return fail(TQ_ERR_UNSUPPORTED, "%s: too many lanes or tokens", what);
    if (int64_t(s->batch) * s->n_kv_heads == 0) return TQ_OK;
    if (!s->k_tail || !s->v_tail || (s->capacity && (!s->k_codes || !s->v_codes || !s->k_scales || !s->v_scales))) return fail(TQ_ERR_INVALID, "%s: null storage", what);
    if (!aligned(s->k_codes, 16) || !aligned(s->v_codes, 16) || !aligned(s->k_tail, 16) || !aligned(s->v_tail, 16) || !aligned(s->k_scales, 4) || !aligned(s->v_scales, 4))
        return fail(TQ_ERR_UNSUPPORTED, "%s: storage must be 16-byte aligned", what);
    return TQ_OK;
}

int blocks_sm_count() {
    static std::atomic<int> n[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int v = n[dev].load();
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
        n[dev].store(v);
    }
    return v;
}

namespace {

struct WriteSide { const void* x; int64_t sb, sh, st; void* codes; float* scales; void* tail; };
struct WriteParams {
    WriteSide side[2];
    int Hkv, lanes, d, block, shift, e4m3;
    int old;                                 // tokens in the tail
    int rest;                                // ... behind the call
    int units;                               // CTAs of a lane: whole blocks, or one where none is full
    int whole;
    int64_t at, blocks_cap;                  // the first block to be filled; blocks of a lane's storage
    int64_t n_new;
};

// Eight values of a row, and eight codes
template <typename E> struct Eight8;
template <> struct Eight8<__half> { uint4 v; };
template <> struct Eight8<__nv_bfloat16> { uint4 v; };
template <> struct Eight8<float> { uint4 v[2]; };
template <typename E> __device__ __forceinline__ Eight8<E> load8(const E* p) { return *reinterpret_cast<const Eight8<E>*>(p); }
template <typename E> __device__ __forceinline__ void store8(E* p, const Eight8<E>& v) { *reinterpret_cast<Eight8<E>*>(p) = v; }
template <typename E> __device__ __forceinline__ float at8(const Eight8<E>& v, int i) { return to_f32<E>(reinterpret_cast<const E*>(&v)[i]); }

// the largest magnitude of eight values, as the bits of the type, and as those of a float32
__device__ __forceinline__ uint32_t largest8(const uint4& v) {
    const uint32_t k = 0x7fff7fffu, z = __vmaxu2(__vmaxu2(v.x & k, v.y & k), __vmaxu2(v.z & k, v.w & k));
    return max(z & 0xffffu, z >> 16);
}
__device__ __forceinline__ uint32_t largest8(const Eight8<__half>& e) { return largest8(e.v); }
__device__ __forceinline__ uint32_t largest8(const Eight8<__nv_bfloat16>& e) { return largest8(e.v); }
__device__ __forceinline__ uint32_t largest8(const Eight8<float>& e) {
    const uint32_t k = 0x7fffffffu;
    return max(max(max(e.v[0].x & k, e.v[0].y & k), max(e.v[0].z & k, e.v[0].w & k)), max(max(e.v[1].x & k, e.v[1].y & k), max(e.v[1].z & k, e.v[1].w & k)));
}
template <typename E> __device__ __forceinline__ uint32_t bits32(uint32_t b) {
    return std::is_same<E, float>::value ? b : std::is_same<E, __half>::value ? __float_as_uint(__half2float(__ushort_as_half(uint16_t(b)))) : b << 16;
}

constexpr int WR_U = 4;                      // vectors of eight values per thread: a CTA has block * d / 32 threads (32 to 1024)

// two float32 at once
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint2 halves_of(uint64_t v) {
    uint2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(r.x), "=r"(r.y) : "l"(v));
    return r;
}

// A CTA works on blocks of (lane, keys or values), gridDim.x apart, the next one's rows on their way in registers while this one is quantised.  Bound by instructions
// as much as by memory: the places of a thread's vectors in a block are the same for all blocks, the maximum is taken on the types' own bits, sums are packed
// (us for 8 x 65,519 tokens a side at d = 128, 402 MB: a CTA per block 110; one after the other with divisions inside 115; so 90; without the divisions 67 = 6.0 TB/s).
// The first block of a lane is the only one that reads the tail, and whoever works on it leaves the rest there, behind its own reads.
// FULL: block * d / 32 is a multiple of 32, so that a thread's vectors are block / 4 rows apart, all of them there.
template <typename E, bool E4M3, bool FULL> __global__ void __launch_bounds__(1024) blocks_write_kernel(const __grid_constant__ WriteParams p) {
    __shared__ uint32_t top[2][32];
    const int per_row = p.d / 8, tid = threadIdx.x, n = p.block * per_row, units = p.units;          // (n: vectors of a block)
    const int row0 = tid / per_row, at = (tid - row0 * per_row) * 8;
    // row and value of this thread's u-th vector of a block; negative: it has none
    auto row_of = [&](int u) { return FULL ? row0 + u * (p.block >> 2) : tid + u * int(blockDim.x) < n ? (tid + u * int(blockDim.x)) / per_row : -1; };
    auto at_of = [&](int u) { return FULL ? at : (tid + u * int(blockDim.x)) % per_row * 8; };
    // units i = (lane, side, block): the next one without a division
    const uint32_t step_ls = gridDim.x / uint32_t(units), step_unit = gridDim.x - step_ls * uint32_t(units);
    uint32_t ls = blockIdx.x / uint32_t(units), unit = blockIdx.x - ls * uint32_t(units);
    const E *src = nullptr;
    E* tail = nullptr;
    int64_t st = 0;
    auto enter = [&]() {
        const uint32_t lane = ls >> 1;
        const bool v = ls & 1;
        const int64_t sb = v ? p.side[1].sb : p.side[0].sb, sh = v ? p.side[1].sh : p.side[0].sh;
        st = v ? p.side[1].st : p.side[0].st;
        int64_t off = int64_t(lane) * sh;
        if (sb != int64_t(p.Hkv) * sh) {                   // (lanes that are not evenly spaced)
            const uint32_t b = lane / uint32_t(p.Hkv);
            off = b * sb + (lane - b * uint32_t(p.Hkv)) * sh;
        }
        src = static_cast<const E*>(v ? p.side[1].x : p.side[0].x) + off;
        tail = static_cast<E*>(v ? p.side[1].tail : p.side[0].tail) + int64_t(lane) * p.block * p.d;
    };
    pdl_wait();
    pdl_trigger();
    Eight8<E> next[WR_U];
    auto load = [&]() {
        const int first = int(unit) * p.block - p.old;     // new token of the block's row 0 (negative: in the tail)
        if (FULL && first >= 0) {
            const E* from = src + ((first + row0) * st + at);
            const int64_t step = (p.block >> 2) * st;
#pragma unroll
            for (int u = 0; u < WR_U; ++u, from += step) next[u] = load8<E>(from);
        } else {
#pragma unroll
            for (int u = 0; u < WR_U; ++u) {
                const int r = row_of(u);
                if (r >= 0) next[u] = load8<E>((first + r < 0 ? tail + r * p.d : src + (first + r) * st) + at_of(u));
            }
        }
    };
    enter();
    if (p.whole > 0) load();
    for (int turn = 0;; turn ^= 1) {
        const uint32_t ls0 = ls, unit0 = unit;
        const E* const src0 = src;
        E* const tail0 = tail;
        const int64_t st0 = st;
        ls += step_ls;
        unit += step_unit;
        if (unit >= uint32_t(units)) { unit -= uint32_t(units); ++ls; }
        const bool more = ls < uint32_t(p.lanes) * 2u;
        if (p.whole > 0) {
            Eight8<E> x[WR_U];
            uint32_t mx = 0;
#pragma unroll
            for (int u = 0; u < WR_U; ++u) {
                x[u] = next[u];
                if (FULL || row_of(u) >= 0) mx = max(mx, largest8(x[u]));      // (magnitudes order like integers, NaN above infinity)
            }
            if (more) {
                enter();
                load();
            }
            mx = __reduce_max_sync(0xffffffffu, mx);
            if ((tid & 31) == 0) top[turn][tid >> 5] = mx;
            __syncthreads();                               // (the maxima of two blocks take turns: nobody writes what another still reads)
            mx = (tid & 31) < int(blockDim.x >> 5) ? top[turn][tid & 31] : 0u;
            mx = bits32<E>(__reduce_max_sync(0xffffffffu, mx));
            const float a = __uint_as_float(mx);
            constexpr float largest = E4M3 ? 448.f : 127.f;
            const bool finite = mx < 0x7f800000u;
            // (127 / A overflows below 4e-37: values that small lose digits, and zeros stay zeros)
            const float inv = !finite || mx == 0u ? 0.f : fminf(__fdiv_rn(largest, a), 3.4028235e38f);
            const int64_t blk = int64_t(ls0 >> 1) * p.blocks_cap + p.at + unit0;
            uint2* out = reinterpret_cast<uint2*>(static_cast<uint8_t*>((ls0 & 1) ? p.side[1].codes : p.side[0].codes) + blk * p.block * p.d) + tid;
            const uint64_t magic2 = two(12582912.f, 12582912.f);
#pragma unroll
            for (int u = 0; u < WR_U; ++u) {
                if (!FULL && row_of(u) < 0) continue;
                uint32_t c[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    // (products one by one: packed ones are contracted with the sums behind them, and a product next to a tie is then rounded once, not twice)
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = __fmul_rn(at8<E>(x[u], 4 * k + j), inv);
                    if (E4M3) {
                        c[k] = e4m3x2_of(y[0], y[1]) | (e4m3x2_of(y[2], y[3]) << 16);
                        if (!finite) c[k] = 0u;            // (a code of its own that is NaN would reach queries that the token is hidden from)
                    } else {
                        // to the nearest integer by adding 1.5 * 2^23 (|y| < 2^22): the low byte of the sum; bytes of two words at a time
                        const uint2 q0 = halves_of(add_two(two(y[0], y[1]), magic2)), q1 = halves_of(add_two(two(y[2], y[3]), magic2));
                        c[k] = __byte_perm(__byte_perm(q0.x, q0.y, 0x0040), __byte_perm(q1.x, q1.y, 0x0040), 0x5410);
                    }
                }
                out[u * blockDim.x] = make_uint2(c[0], c[1]);
            }
            if (tid == 0) ((ls0 & 1) ? p.side[1].scales : p.side[0].scales)[blk] = finite ? __fdiv_rn(a, largest) : __uint_as_float(0x7fffffffu);
        } else if (more) {
            enter();
        }
        if (unit0 == 0) {
            // the rest: behind the whole blocks from row 0 on, or behind what the tail holds
            const int to = p.whole > 0 ? 0 : p.old, rows = p.rest - to;
            const int64_t t0 = p.whole > 0 ? p.n_new - p.rest : 0;
            for (int i = tid; i < rows * per_row; i += blockDim.x) {
                const int r = i / per_row, c = (i - r * per_row) * 8;
                store8<E>(tail0 + int64_t(to + r) * p.d + c, load8<E>(src0 + (t0 + r) * st0 + c));
            }
        }
        if (!more) break;
    }
}

struct ReadParams {
    const uint8_t* codes[2]; const float* scales[2]; const void* tail[2]; void* out[2];
    int d, block, shift, e4m3, dtype, out_dtype;
    uint32_t blocks_per_lane, n, n8;         // vectors of 16 values of a lane, of them in blocks
    int64_t cap, length;
};
constexpr int RD_T = 256, RD_U = 4;

template <typename O> __device__ __forceinline__ uint32_t pair_of(float a, float b);
template <> __device__ __forceinline__ uint32_t pair_of<__half>(float a, float b) { return pack_h2(a, b); }
template <> __device__ __forceinline__ uint32_t pair_of<__nv_bfloat16>(float a, float b) { return pack_bf2(a, b); }

// sixteen values of the tail, of any type, as float32
__device__ __forceinline__ void tail16(const void* t, int dtype, int64_t i, float (&x)[16]) {
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = load_as_f32(t, dtype, i + k);
}
template <typename O> __device__ __forceinline__ void store16(O* o, const float (&x)[16]) {
    if constexpr (sizeof(O) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) reinterpret_cast<float4*>(o)[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = pair_of<O>(x[2 * k], x[2 * k + 1]);
        reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

template <typename O> __global__ void __launch_bounds__(RD_T) blocks_read_kernel(const __grid_constant__ ReadParams p) {
    const uint32_t ls = blockIdx.x / p.blocks_per_lane, blk = blockIdx.x - ls * p.blocks_per_lane, per_row = uint32_t(p.d) / 16;
    const int side = ls & 1;
    const int64_t lane = ls >> 1;
    const uint8_t* codes = p.codes[side] + lane * p.cap * p.d;
    const float* scales = p.scales[side] + lane * (p.cap >> p.shift);
    O* out = static_cast<O*>(p.out[side]) + lane * p.length * p.d;
    pdl_wait();
    pdl_trigger();
    uint4 c[RD_U];
    float s[RD_U];
#pragma unroll
    for (int u = 0; u < RD_U; ++u) {
        const uint32_t i = (blk * RD_U + u) * RD_T + threadIdx.x;
        if (i < p.n8) {
            c[u] = reinterpret_cast<const uint4*>(codes)[i];
            s[u] = scales[(i / per_row) >> p.shift];
        }
    }
#pragma unroll
    for (int u = 0; u < RD_U; ++u) {
        const uint32_t i = (blk * RD_U + u) * RD_T + threadIdx.x;
        if (i >= p.n) continue;
        float x[16];
        if (i < p.n8) {
            const uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const uint32_t byte = (w[k >> 2] >> (8 * (k & 3))) & 255u;
                x[k] = (p.e4m3 ? e4m3_to_f32(uint8_t(byte)) : float(int8_t(byte))) * s[u];
            }
        } else {
            tail16(p.tail[side], p.dtype, lane * p.block * p.d + int64_t(i - p.n8) * 16, x);
        }
        store16<O>(out + int64_t(i) * 16, x);
    }
}

}  // namespace
}  // namespace tq

extern "C" int tq_blocks_write(const tq_block_store* s, const tq_new_rows* k_new, const tq_new_rows* v_new, int64_t n_new, void* stream) {
    using namespace tq;
    if (int rc = check_store(s, "tq_blocks_write")) return rc;
    if (n_new < 0 || !k_new || !v_new) return fail(TQ_ERR_INVALID, "tq_blocks_write: bad new tokens");
    const int lanes = s->batch * s->n_kv_heads;
    if (n_new == 0 || lanes == 0) return TQ_OK;
    if (s->length + n_new >= (1 << 30)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_write: too many tokens");
    WriteParams p{};
    p.Hkv = s->n_kv_heads; p.lanes = lanes; p.d = s->d; p.block = s->block; p.shift = log2_of(s->block); p.e4m3 = s->code_type == TQ_CODE_E4M3;
    p.old = int(s->length % s->block);
    p.whole = int((p.old + n_new) / s->block);
    p.rest = int((p.old + n_new) % s->block);
    p.at = s->length / s->block; p.blocks_cap = s->capacity / s->block; p.n_new = n_new;
    if (p.at + p.whole > p.blocks_cap)
        return fail(TQ_ERR_INVALID, "tq_blocks_write: %lld tokens and %lld more in storage for %lld", (long long)s->length, (long long)n_new, (long long)s->capacity);
    p.units = std::max(p.whole, 1);
    const int es = s->dtype == TQ_F32 ? 4 : 2;
    for (int i = 0; i < 2; ++i) {
        const tq_new_rows& r = i ? *v_new : *k_new;
        if (!r.x) return fail(TQ_ERR_INVALID, "tq_blocks_write: null rows");
        if (!aligned(r.x, 16) || (r.sb * es) % 16 || (r.sh * es) % 16 || (r.st * es) % 16) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_write: rows must be 16-byte aligned");
        p.side[i] = WriteSide{r.x, r.sb, r.sh, r.st, i ? s->v_codes : s->k_codes, i ? s->v_scales : s->k_scales, i ? s->v_tail : s->k_tail};
    }
    const int64_t blocks = int64_t(p.units) * lanes * 2;
    if (blocks >= (int64_t(1) << 31)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_write: too many blocks");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    const int threads = (s->block * s->d / (8 * WR_U) + 31) / 32 * 32;
    const bool full = s->block * s->d / (8 * WR_U) == threads;
    // as many CTAs as the SMs hold (64 registers a thread)
    const int64_t room = int64_t(blocks_sm_count()) * std::min(32, 1024 / threads);
    cfg.gridDim = dim3(unsigned(std::min(blocks, room)));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto pick = [&](auto* full8, auto* full_i, auto* any8, auto* any_i) { cudaLaunchKernelEx(&cfg, full ? (p.e4m3 ? full8 : full_i) : (p.e4m3 ? any8 : any_i), p); };
    if (s->dtype == TQ_F16) pick(blocks_write_kernel<__half, true, true>, blocks_write_kernel<__half, false, true>, blocks_write_kernel<__half, true, false>, blocks_write_kernel<__half, false, false>);
    else if (s->dtype == TQ_BF16) pick(blocks_write_kernel<__nv_bfloat16, true, true>, blocks_write_kernel<__nv_bfloat16, false, true>, blocks_write_kernel<__nv_bfloat16, true, false>, blocks_write_kernel<__nv_bfloat16, false, false>);
    else pick(blocks_write_kernel<float, true, true>, blocks_write_kernel<float, false, true>, blocks_write_kernel<float, true, false>, blocks_write_kernel<float, false, false>);
    return check_launch("tq_blocks_write");
}

extern "C" int tq_blocks_read(const tq_block_store* s, void* k_out, void* v_out, int out_dtype, void* stream) {
    using namespace tq;
    if (int rc = check_store(s, "tq_blocks_read")) return rc;
    if (!dtype_ok(out_dtype)) return fail(TQ_ERR_INVALID, "tq_blocks_read: bad result type %d", out_dtype);
    const int64_t lanes = int64_t(s->batch) * s->n_kv_heads;
    if (lanes == 0 || s->length == 0) return TQ_OK;
    if (!k_out || !v_out) return fail(TQ_ERR_INVALID, "tq_blocks_read: null results");
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_read: results must be 16-byte aligned");
    const int64_t n = s->length * (s->d / 16);
    if (n >= (int64_t(1) << 31)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_read: too many tokens");
    ReadParams p{};
    p.codes[0] = static_cast<const uint8_t*>(s->k_codes); p.codes[1] = static_cast<const uint8_t*>(s->v_codes);
    p.scales[0] = s->k_scales; p.scales[1] = s->v_scales;
    p.tail[0] = s->k_tail; p.tail[1] = s->v_tail; p.out[0] = k_out; p.out[1] = v_out;
    p.d = s->d; p.block = s->block; p.shift = log2_of(s->block); p.e4m3 = s->code_type == TQ_CODE_E4M3; p.dtype = s->dtype;
    p.n = uint32_t(n); p.n8 = uint32_t(s->length / s->block * s->block * (s->d / 16));
    p.cap = s->capacity; p.length = s->length;
    p.blocks_per_lane = (p.n + RD_T * RD_U - 1) / (RD_T * RD_U);
    const int64_t blocks = int64_t(p.blocks_per_lane) * lanes * 2;
    if (blocks >= (int64_t(1) << 31)) return fail(TQ_ERR_UNSUPPORTED, "tq_blocks_read: too many tokens");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(RD_T);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (out_dtype == TQ_F16) cudaLaunchKernelEx(&cfg, blocks_read_kernel<__half>, p);
    else if (out_dtype == TQ_BF16) cudaLaunchKernelEx(&cfg, blocks_read_kernel<__nv_bfloat16>, p);
    else cudaLaunchKernelEx(&cfg, blocks_read_kernel<float>, p);
    return check_launch("tq_blocks_read");
}
