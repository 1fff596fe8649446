// Declarations shared by the kernels of the 8-bit block cache.
#pragma once

#include "decode_dev.cuh"

namespace tq {

constexpr int BLOCKS_MAX_D = 256;

inline bool block_ok(int n) { return n == 16 || n == 32 || n == 64 || n == 128; }
inline int log2_of(int n) { return 31 - __builtin_clz(unsigned(n)); }
// What every entry point of the cache asks of its storage; `what` opens the error's text
int check_store(const tq_block_store* s, const char* what);
int blocks_sm_count();

// blocks_attend.cu: float32 tokens and head dims without a kernel of their own; one new token, and a few, per sequence
// blocks_fa.cu: many query rows per lane
struct BlockAttendParams {
    const uint8_t *kc, *vc;                  // codes
    const float *ks, *vs;                    // scales
    const void *kt, *vt;                     // tails
    void *kt_w, *vt_w;                       // tails, writable (append)
    const void *kn, *vn;                     // the appended token's rows, or null
    int64_t kn_sb, kn_sh, vn_sb, vn_sh;
    const void* q;
    int64_t q_sb, q_sh, q_st;
    void* out;
    int dtype, e4m3;
    int B, Hq, Hkv, G, D, Tq;
    int block, shift;                        // tokens of a block, log2 of that
    int64_t cap;                             // tokens of a lane's codes; cap >> shift scales
    int n8, total;                           // tokens in blocks; all tokens, the appended one included
    int window, sinks;                       // window: INT_MAX / 2 without one
    float scale_log2;                        // scale * log2(e)
    float* part;                             // workspace
    size_t room;                             // its bytes; all there may be where only the need is asked
};

int launch_blocks_plain(const BlockAttendParams& p, cudaStream_t s);
double blocks_split_us(const BlockAttendParams& p);      // what a call is expected to cost in blocks_attend.cu's kernel
bool blocks_fa_takes(const BlockAttendParams& p);
size_t blocks_fa_workspace(const BlockAttendParams& p);
int blocks_fa_choice(const BlockAttendParams& p);        // TQ_BLOCKS_FUSED ... TQ_BLOCKS_EXPANDED_CUT
int launch_blocks_fa(const BlockAttendParams& p, cudaStream_t s);

// The first token that some query sees through its window, and how many sink tokens lie before it
struct Visible { int low, sinks; };
inline __host__ __device__ Visible visible_of(int total, int t_q, int window, int sinks) {
    const int first = total - t_q, low = first - window + 1 > 0 ? first - window + 1 : 0;
    return Visible{low, sinks < low ? sinks : low};
}

__device__ __forceinline__ uint32_t e4m3x2_of(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(c)));
    return __half2float(__ushort_as_half(uint16_t(h & 0xffffu)));
}

__device__ __forceinline__ void ld_codes(uint4& x, const uint8_t* p) {
    asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t at, uint4 x) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
// four codes as two pairs of fp16.  int8: biased by 128 they are the low bytes of 1024 + code + 128
template <bool E4M3> __device__ __forceinline__ void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t k = 0x64806480u;
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(k));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(k));
    }
}

}  // namespace tq
