// Gated feed-forward block at every point of a field, forward and backward, on the tensor cores (tcgen05).
//
//   g = W_gate x + b_gate,  u = W_up x + b_up,  h = act(g) u,  y = W_down h + b_down
//
// x [B, C, P], hidden width H, y [B, O, P]; act is SiLU or the exact GELU.  Backward, with e = dL/dy:
//
//   f = W_down^T e,  dg = f u act'(g),  du = f act(g),  dL/dx = W_gate^T dg + W_up^T du,
//   dL/dW_gate = dg x^T,  dL/dW_up = du x^T,  dL/dW_down = e h^T (sums over all points), biases: row sums.
//
// Both passes are one kernel shape (k_block).  A tile is 128 points (the MMA's M); the hidden width is walked in
// chunks of NH.  A job is one chunk of one tile:
//   first product   D1 = [g | u] (backward: [g | u | f])   A = x (and e) from shared memory, B = weights
//   middle          the epilogue warps read D1, apply the activation and write h (backward: dg, du) back into the
//                   same columns of tensor memory as the next A operand -- h never leaves the SM in the forward
//   second product  D2 += h W_down^T (backward: dg W_gate + du W_up), A from tensor memory
// and after a tile's last chunk (fp32: after every kRunSteps steps) D2 goes out.  Two or three D1 buffers take turns, so the
// tensor core works on the next jobs' first products while the epilogue warps work on a job; a tile's D2 is read after the
// next tile's first middle.
//
// Operands.  16-bit fields multiply as they are (products exact, fp32 sums); h, dg and du go into their products in two
// 16-bit parts (Mid), and into the weights' gradients in two bf16 parts or in fp32 (Scratch).  fp32 values are split into three
// bf16 parts, v = a + b + c to within 2^-26 |v|, and six of the nine products are summed (the three left out are
// below 2^-26): near fp32 accuracy at the cost of six 16-bit MMAs, the same tensor time as three tf32 passes on a
// hi / lo split but three quarters of its shared memory, and 2^-26 instead of 2^-21.  The tensor core adds to its
// accumulator with truncation, about 2^-25 of it towards zero every time, so the five smaller products, 2^-8 of the
// first and less, are kept from the large accumulator: the second product gives them columns of their own (D2c,
// added at the end), the first product adds them before the large one, piece by piece.  (All six into one
// accumulator: dL/dx was 4.7e-6 off at 128 channels, hidden 200.)  From the second piece on they meet a large D1 all the
// same, for which tensor memory has no second set of columns: outputs are 0.5 to 1.1e-6 of their size off float64 at up to
// 64 channels, 1.8e-6 at 128 and 3.6e-6 at 256 (fp32 products: 0.3 to 0.9e-6).  fp16: h, and dg and du on their way into
// dL/dx, have fp16's range and its smallest step, 2^-24.  An e4m3 field is widened exactly and its point's scale multiplies
// the accumulator.
//
// The points of a channel are contiguous and the MMA wants a point's channels contiguous (K-major core matrices of
// 8 rows x 16 bytes): a producer thread loads 8 channels x 4 points with one wide load a channel and writes four
// 16-byte rows, so the transposition is a choice of registers.  The core matrices of 8-row groups lie 272 bytes
// apart instead of 256: the rows that eight neighbouring threads write then fall into eight different 16-byte
// columns of the banks.  Weights are packed once a call (k_pack) into images that a bulk copy brings into shared
// memory whole; they stay there for the whole kernel when they fit, and stream through a ring otherwise.
//
// The weight gradients contract over points, which are contiguous in every operand: k_wgrad reads dg, du, h,
// x and e, all by tensor copies, splits the points over the CTAs and leaves partial sums that k_finish adds in a fixed
// order.  k_block leaves dg, du and h in a scratch [tile][rows][128 points] (with rows as long as the slab every store
// went to a page of its own, 100 cycles each), and x and e too, unless their samples are whole tiles on aligned rows
// that a tensor copy can read in place.  Because of the truncation a long sum is cut: every kPromote pieces the
// epilogue warps add the accumulator (fp32: and the smaller products' own) to registers.
// The scratch is made and consumed slab by slab.
//
// Measured on B200.  fp32, 64 / 128 / 64 (channels, hidden, out): the forward of 2^21 points takes 500 us (600 in a long
// run, at the power cap's 1.6 GHz), where the bytes take 166 us and six 16-bit products 371 us at the measured peaks.
// It is bound by the MMA warp, which never waits: the first product's MMAs take 105 cycles each instead of the 68 of
// their arithmetic, both operands coming from shared memory, the second one's (N = 64) 50; the middle takes 1650 cycles
// of a job's 4050.  A third D1 buffer, more weights or pieces of x in flight, or MMAs issued in blocks changed nothing.
// 16-bit types are bound by the middle (800 cycles for 16 hidden channels of a warp's points; exponentials, reciprocals
// and conversions): bf16 128 / 384 / 128 on 32 fields of 85 x 85, rows not aligned, 153 us forward and 684 us backward
// (products alone: 41 and 110 us); 64 / 128 / 64 on 2^20 points 182 and 915 us, fp16 184 and 1052.  In the backward the
// scratch's stores lengthen the middle (to 4400 cycles a job with dg, du and h rounded to one part, whose bytes were half:
// 484 and 557 us), and k_wgrad reads it at 4.6 TB/s.  Pairs of CTAs (cta_group::2, half of the weights in each) ran slower at nearly all
// sizes (fp32 forward above 548 us, bf16 32 / 32 / 32 121 us against 70).
//
// Every wait is bounded: on expiry the kernel records NOP_DEVICE_MMA_TIMEOUT in the status word, all roles leave
// their loops, copies and MMAs in flight are waited for (bounded) and the tensor memory is freed.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "mix_tc.cuh"

namespace nop {
namespace gated {

constexpr int TP = 128;                       // points a tile
constexpr int kSmem = 227 * 1024;
constexpr int kAGroup = 272;                  // bytes between 8-row groups of an A image
constexpr int kMaxA = 8, kMaxB = 8;           // ring slots at most

__host__ __device__ constexpr int up16(int v) { return (v + 15) & ~15; }
__host__ __device__ constexpr int imin(int a, int b) { return a < b ? a : b; }

// Operand form of a field type: images an operand has, elements of K a ring piece has
template <class T> struct Form {
    static constexpr int SPL = 1, KC = 64;
    static constexpr uint32_t kFmt = 1;       // bf16
};
template <> struct Form<float> {
    static constexpr int SPL = 3, KC = 32;
    static constexpr uint32_t kFmt = 1;
};
template <> struct Form<__half> {
    static constexpr int SPL = 1, KC = 64;
    static constexpr uint32_t kFmt = 0;
};
// the products of the images, the large one first: (A image, B image)
template <int SPL> struct Passes {
    static constexpr int N = SPL == 1 ? 1 : 6;
    __device__ static constexpr int a(int i) { return i == 2 || i == 3 ? 1 : i == 5 ? 2 : 0; }
    __device__ static constexpr int b(int i) { return i == 1 || i == 3 ? 1 : i == 4 ? 2 : 0; }
};

// What the backward's scratch holds dg, du and h in: fp32 values of fp32 and fp16 fields (a gradient below 2^-24 or above
// 65504 is not lost on its way into a sum), two bf16 parts of bf16 fields, which multiply as they lie.  Rounded once to
// 16 bits they put the weights' gradients off by 1.4 times the result's own rounding.
template <class T> struct Scratch {
    using type = float;
    static constexpr int PARTS = 1;
};
template <> struct Scratch<__nv_bfloat16> {
    using type = __nv_bfloat16;
    static constexpr int PARTS = 2;
};

// Warps of k_block.
constexpr int kEpi = 8;                       // 0..7: middle and output
constexpr int kProd = 4;                      // 8..11: x (and e) into shared memory
constexpr int kMma = kEpi + kProd;            // 12: MMA issue
constexpr int kLoad = kMma + 1;               // 13: weight copies
constexpr int kThreads = 32 * (kLoad + 1);    // 14 warps: 128 registers a thread

// fp32: K steps (of 16 hidden channels) that D2 runs before it is added to the output.  Every step truncates D2 by about
// 2^-25 of it, always towards zero, so a sum over a whole wide hidden layer drifts: 1.7e-5 in y and 3.8e-5 in dL/dx at a
// width of 16384, where 32 steps are below 1e-6.  16-bit results are rounded by far more.
constexpr int kRunSteps = 32;

struct Plan {
    int C, H, O;               // channels of x, hidden width, channels of y
    int Kx, Ky;                // padded K of the first products (Ky: backward only, 0 otherwise)
    int cols, col0;            // channels of this launch's output, the first of them
    int N2;                    // padded columns of D2
    int n_d1, n_d2;            // D1 buffers (jobs in flight), D2 buffers
    int NH, nJ;                // chunk width, chunks
    int per, runs;             // chunks that D2 runs before it goes out, times it goes out a tile
    int nKx, nKy, nH;          // ring pieces: of x, of e, of a chunk in the second product
    int na, nb;                // ring slots (nb: streaming)
    int reuse;                 // 1: a tile's A pieces stay in the ring for all its chunks
    int resident;              // 1: all weight images stay in shared memory
    int a_slot, b_slot;        // bytes
    int job_bytes;             // packed weight bytes of one chunk
    int vec_smem;              // 1: the biases have a copy in shared memory
    int o_a, o_b, o_vec, o_bar, smem;
};

struct Params {
    const void* x;
    const void* gy;            // backward: e
    const float* scale;        // e4m3 x: one a point
    const char* packed;
    const float* bias;         // the biases of g, u and (forward) of the output: fp32, padded with zeros
    void* out;                 // y, or dL/dx (may be NULL)
    void* z;                   // backward: [tile][z_rows][128] dg, du, h (their second parts) (x, e) (may be NULL)
    int z_rows;                // 3 H PARTS, or that and C + O
    uint32_t P, points;        // a sample's points, all points
    uint32_t p_mul, p_shift;   // n / P = n p_mul >> p_shift for n < 2^31
    int tile0, tiles;          // tiles of this launch
    int vec;                   // 4 points a load
    Plan pl;
};

// The sample of point n.  A division by a run-time number costs some 100 cycles and several stood in every tile's
// path: with s = ceil(log2 P) and m = ceil(2^(31 + s) / P) < 2^32, m P exceeds 2^(31 + s) by less than 2^s, so
// n m / 2^(31 + s) exceeds n / P by less than 1 / P for n < 2^31 and has the same whole part.
__device__ __forceinline__ uint32_t sample_of(const Params& p, uint32_t n) {
    return (uint32_t)(((uint64_t)n * p.p_mul) >> p.p_shift);
}

__host__ __device__ inline int piece_k(int K, int KC, int kc) { return imin(KC, K - kc * KC); }

// ------------------------------------------------------------------------------------------------
// device helpers
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t desc_of(uint32_t addr, int sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ uint32_t idesc_of(uint32_t fmt, int N) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(TP >> 4) << 24);
}
// One lane of the (converged) warp.  The MMA warp runs its loops with all lanes and only predicates the MMAs and
// commits on it: its descriptors and addresses then stay in uniform registers.  With the loops inside a one-lane
// branch every MMA cost its warp 105 to 120 cycles, more than the tensor core needs for most of them.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%6, %6, %6, %6}, p;\n\t}"
        :
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u), "r"(leader), "r"(0)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%6, %6, %6, %6}, p;\n\t}"
        :
        : "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u), "r"(leader), "r"(0)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_u32(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// the registers are operands, so no use of them moves above the wait
__device__ __forceinline__ void wait_ld(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                   "+f"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// bounded wait (tc::mbar_wait) that first asks without reading the clock
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(tc::smem_u32(bar)), "r"(parity)
        : "memory");
    return done || tc::mbar_wait(bar, parity, abort);
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(bytes)
                 : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two neighbouring K elements as one word of each image.  Pairs of values go through packed fp32 arithmetic
// wherever there is some: the epilogue warps are bound by their instruction count.
template <class T> __device__ __forceinline__ void images(float2 v, uint32_t (&w)[Form<T>::SPL]);
template <> __device__ __forceinline__ void images<__nv_bfloat16>(float2 v, uint32_t (&w)[1]) {
    w[0] = tc::pack_bf16(v.x, v.y);
}
template <> __device__ __forceinline__ void images<__half>(float2 v, uint32_t (&w)[1]) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    w[0] = *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ void images<float>(float2 v, uint32_t (&w)[3]) {
    // v = a + b + c, each part the rounding of what is left (the differences are exact)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        w[i] = tc::pack_bf16(v.x, v.y);
        if (i < 2) v = __ffma2_rn(make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)),
                                  make_float2(-1.f, -1.f), v);
    }
}

// The second product's A operand, which the middle makes from fp32 values: the three parts of fp32, and for a 16-bit
// type the rounded value and the rounding of what is left.  With one rounding of h the output was off by up to 1.5
// times its own rounding; the second MMA a step costs nothing that shows, the middle being the longer part.
template <class T> struct Mid {
    static constexpr int N = 2;
};
template <> struct Mid<float> {
    static constexpr int N = 3;
};
template <class T> __device__ __forceinline__ void mid_images(float2 v, uint32_t (&w)[Mid<T>::N]) {
    if constexpr (std::is_same<T, float>::value) {
        images<T>(v, w);
    } else {
        uint32_t t[1];
        images<T>(v, t);
        w[0] = t[0];
        float2 back;
        if constexpr (std::is_same<T, __half>::value) back = __half22float2(*reinterpret_cast<const __half2*>(&t[0]));
        else back = make_float2(__uint_as_float(t[0] << 16), __uint_as_float(t[0] & 0xFFFF0000u));
        images<T>(__ffma2_rn(back, make_float2(-1.f, -1.f), v), t);
        w[1] = t[0];
    }
}

__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// two reciprocals for one special-function operation, which bound the middle (16 a cycle and SM): 1 / (x y) times the
// other one
__device__ __forceinline__ float2 rcp2(float2 v) { return __fmul2_rn(both(rcp_approx(v.x * v.y)), make_float2(v.y, v.x)); }

// act(g) and act'(g) of two values.  SiLU: g s, s + g s (1 - s), s = 1 / (1 + exp(-g)), where 1 - s = exp(-g) s: a
// subtraction would leave the reciprocal's last bit, which g multiplies (slope 1e-3 off at g = 1e4).  GELU: g P(g),
// P(g) + g p(g) with the normal distribution function P from erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2),
// t = 1 / (1 + q x), Abramowitz & Stegun, Handbook of Mathematical Functions (1964), eq. 7.1.26 (|error| <= 1.5e-7);
// its exponential is also the density's.  Reciprocal and exponential are the special-function unit's (2^-22 or so).
template <bool GELU>
__device__ __forceinline__ float2 activation(float2 g, float2& slope) {
    if (!GELU) {
        // g is held at -60 ln 2, where |silu| < 4e-17: the exponential is 2^60 there, and the product of two is finite
        const float2 c = make_float2(max_nan(g.x, -41.588830834f), max_nan(g.y, -41.588830834f));
        const float2 t = __fmul2_rn(c, both(-1.4426950408889634f));
        const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
        const float2 s = rcp2(__fadd2_rn(e, both(1.f)));
        const float2 a = __fmul2_rn(c, s);
        slope = __ffma2_rn(a, __fmul2_rn(e, s), s);
        return a;
    }
    // |g| = sqrt(2) times erfc's argument; the exponential is zero long before 64, and the product of two denominators
    // has to be finite (a neighbour of a gate of 3e38 came out as if it were saturated)
    const float2 x = make_float2(fminf(fabsf(g.x), 64.f), fminf(fabsf(g.y), 64.f));
    const float2 d = __ffma2_rn(x, both(0.3275911f * 0.70710678118654752f), both(1.f));
    const float2 t = rcp2(d);
    const float2 q = __fmul2_rn(__fmul2_rn(g, g), both(-0.5f * 1.4426950408889634f));
    const float2 e = make_float2(exp2_approx(q.x), exp2_approx(q.y));
    float2 s = __ffma2_rn(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
    s = __ffma2_rn(t, s, both(0.5f * 1.421413741f));
    s = __ffma2_rn(t, s, both(0.5f * -0.284496736f));
    s = __ffma2_rn(t, s, both(0.5f * 0.254829592f));
    const float2 tail = __fmul2_rn(__fmul2_rn(s, t), e);   // P(-|g|)
    const float2 cdf = make_float2(g.x < 0.f ? tail.x : 1.f - tail.x, g.y < 0.f ? tail.y : 1.f - tail.y);
    slope = __ffma2_rn(__fmul2_rn(g, both(0.3989422804014327f)), e, cdf);
    return __fmul2_rn(g, cdf);
}

// ------------------------------------------------------------------------------------------------
// weights -> images
// ------------------------------------------------------------------------------------------------
// One thread packs 8 elements of K of one row of one piece.  Chunk j's pieces follow one another: the first
// product's (rows: NH of W_gate, NH of W_up; K: channels of x), backward the f product's (rows: NH hidden; K:
// channels of e, from W_down), then the second product's (forward: rows O, K hidden, from W_down; backward: rows C,
// K hidden, from W_gate and then from W_up).
template <class T, bool BWD>
__global__ void __launch_bounds__(256)
k_pack(Plan pl, const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ wd, const T* __restrict__ bg,
       const T* __restrict__ bu, const T* __restrict__ bd, char* __restrict__ packed, float* __restrict__ vec) {
    constexpr int SPL = Form<T>::SPL, KC = Form<T>::KC;
    const int hid = pl.NH * pl.nJ;
    const int stride = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
    for (int i = first; i < 2 * hid + pl.N2; i += stride) {
        const int k = i < hid ? i : i < 2 * hid ? i - hid : i - 2 * hid;
        const T* b = i < hid ? bg : i < 2 * hid ? bu : bd;
        const int n = i < 2 * hid ? pl.H : (BWD ? 0 : pl.cols);
        vec[i] = b && k < n ? to_f(b[i < 2 * hid ? k : pl.col0 + k]) : 0.f;
    }
    const int r1 = 2 * pl.NH, c1 = r1 * (pl.Kx / 8), c2 = BWD ? pl.NH * (pl.Ky / 8) : 0;
    const int c3 = pl.N2 * (pl.NH / 8), per = c1 + c2 + (BWD ? 2 : 1) * c3;
    for (int i = first; i < per * pl.nJ; i += stride) {
        const int j = i / per;
        int c = i % per, off = j * pl.job_bytes;
        int rows, K, part;
        if (c < c1) {
            part = 0;
            rows = r1;
            K = pl.Kx;
        } else if (c < c1 + c2) {
            part = 1;
            off += c1 * 16 * SPL;
            c -= c1;
            rows = pl.NH;
            K = pl.Ky;
        } else {
            off += (c1 + c2) * 16 * SPL;
            c -= c1 + c2;
            part = 2;
            if (c >= c3) {
                c -= c3;
                off += c3 * 16 * SPL;
                part = 3;
            }
            rows = pl.N2;
            K = pl.NH;
        }
        const int row = c % rows, k8 = c / rows;            // neighbouring threads: neighbouring rows
        const int kc = k8 / (KC / 8), ch = k8 % (KC / 8), pw = piece_k(K, KC, kc);
        off += rows * kc * KC * 2 * SPL;                     // the pieces before this one are full
        off += (ch >> 1) * (rows * 32) + (row >> 3) * 256 + (ch & 1) * 128 + (row & 7) * 16;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int k = k8 * 8 + e;
            float w = 0.f;
            if (part == 0) {
                const int h = j * pl.NH + (row < pl.NH ? row : row - pl.NH);
                if (h < pl.H && k < pl.C) w = to_f((row < pl.NH ? wg : wu)[(int64_t)h * pl.C + k]);
            } else if (part == 1) {
                const int h = j * pl.NH + row;
                if (h < pl.H && k < pl.O) w = to_f(wd[(int64_t)k * pl.H + h]);
            } else {
                const int h = j * pl.NH + k;
                if (!BWD) {
                    if (h < pl.H && row < pl.cols) w = to_f(wd[(int64_t)(pl.col0 + row) * pl.H + h]);
                } else if (h < pl.H && row < pl.cols) {
                    w = to_f((part == 2 ? wg : wu)[(int64_t)h * pl.C + pl.col0 + row]);
                }
            }
            v[e] = w;
        }
        uint32_t img[4][SPL];
#pragma unroll
        for (int e = 0; e < 4; ++e) images<T>(make_float2(v[2 * e], v[2 * e + 1]), img[e]);
#pragma unroll
        for (int s = 0; s < SPL; ++s)
            *reinterpret_cast<uint4*>(packed + off + s * rows * pw * 2) =
                make_uint4(img[0][s], img[1][s], img[2][s], img[3][s]);
    }
}

// ------------------------------------------------------------------------------------------------
// x / e -> A images
// ------------------------------------------------------------------------------------------------
// 8 channels x 4 points as loaded: 16-bit and fp32 fields two or four words a channel, e4m3 one
template <class IN> struct Item {
    static constexpr int W = (int)sizeof(IN);  // words a channel
    uint32_t w[8 * W];
};

// A lane's 4 points are 4 lane .. 4 lane + 3 of the tile, but lane, lane + 32, ... of an fp32 field whose rows are
// not aligned (its single loads are then a line each).
template <class IN> __device__ __forceinline__ bool neighbours(bool vec) { return vec || sizeof(IN) < 4; }

// The 4 points one by one, whatever their samples; into r as an Item's words
template <class IN>
__device__ __forceinline__ void load_singly(uint32_t* r, int stride, const IN* __restrict__ src, int C, int c0,
                                            uint32_t n0, int lane, const Params& p) {
    constexpr int W = Item<IN>::W;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < W; ++i) r[e * stride + i] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t n = n0 + (W < 4 ? 4 * lane + i : lane + 32 * i);
        if (n >= p.points) continue;
        const uint32_t b = sample_of(p, n);
        const IN* s = src + (int64_t)b * C * p.P + (n - b * p.P) + (int64_t)c0 * p.P;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (c0 + e >= C) continue;
            const IN* a = s + (int64_t)e * p.P;
            if constexpr (W == 4) r[e * stride + i] = __ldg(reinterpret_cast<const uint32_t*>(a));
            else if constexpr (W == 2)
                r[e * stride + i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(a)) << (16 * (i & 1));
            else
                r[e * stride] |= (uint32_t)__ldg(reinterpret_cast<const uint8_t*>(a)) << (8 * i);
        }
    }
}

template <class IN>
__device__ __forceinline__ void load_item(uint32_t* r, const IN* __restrict__ src, int C, int c0, uint32_t n0, int lane,
                                          const Params& p) {
    constexpr int W = Item<IN>::W;
    if (!p.vec) {
        load_singly<IN>(r, W, src, C, c0, n0, lane, p);
        return;
    }
    const uint32_t n = n0 + 4 * lane;
    const bool ok = n < p.points;
    const uint32_t b = ok ? sample_of(p, n) : 0;
    const IN* s = src + (int64_t)b * C * p.P + (ok ? n - b * p.P : 0) + (int64_t)c0 * p.P;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool in = ok && c0 + e < C;
        const IN* a = s + (int64_t)e * p.P;
        if constexpr (W == 4) {
            const uint4 q = in ? __ldg(reinterpret_cast<const uint4*>(a)) : make_uint4(0, 0, 0, 0);
            r[4 * e] = q.x;
            r[4 * e + 1] = q.y;
            r[4 * e + 2] = q.z;
            r[4 * e + 3] = q.w;
        } else if constexpr (W == 2) {
            const uint2 q = in ? __ldg(reinterpret_cast<const uint2*>(a)) : make_uint2(0, 0);
            r[2 * e] = q.x;
            r[2 * e + 1] = q.y;
        } else {
            r[e] = in ? __ldg(reinterpret_cast<const uint32_t*>(a)) : 0;
        }
    }
}

// A narrow field on rows of any alignment: a channel's 4 values lie in two aligned words of 4 values, which are loaded
// as they are and cut when the item is used (cut_item) -- combined here, they would make the producer wait for every
// load.  Returns the first channel's offset in its word, or 8 where the words would leave the field or the points are
// not of one sample, and the values have been loaded one by one.
template <class IN>
__device__ __forceinline__ uint32_t load_around(uint32_t* r, const IN* __restrict__ src, int C, int c0, uint32_t n0,
                                                int lane, const Params& p) {
    constexpr int W = Item<IN>::W, N = 4 * W;
    const uint32_t n = n0 + 4 * lane;
    const uint32_t b = n < p.points ? sample_of(p, n) : 0, o = n - b * p.P;
    const char* first = reinterpret_cast<const char*>(src + (int64_t)b * C * p.P + o + (int64_t)c0 * p.P);
    const char *begin = reinterpret_cast<const char*>(src), *end = begin + (int64_t)p.points * C * W;
    auto word = [&](int e) {
        return reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(first + (int64_t)e * p.P * W) & ~(uintptr_t)(N - 1));
    };
    const int last = imin(8, C - c0) - 1;
    if (last < 0 || n + 3 >= p.points || o + 3 >= p.P || word(0) < begin || word(last) + 2 * N > end) {
        load_singly<IN>(r, 2 * W, src, C, c0, n0, lane, p);
        return 8;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (W == 2) {
            const uint2* a = reinterpret_cast<const uint2*>(word(e));
            const uint2 q = e <= last ? __ldg(a) : make_uint2(0, 0), t = e <= last ? __ldg(a + 1) : make_uint2(0, 0);
            r[4 * e] = q.x;
            r[4 * e + 1] = q.y;
            r[4 * e + 2] = t.x;
            r[4 * e + 3] = t.y;
        } else if constexpr (W == 1) {
            const uint32_t* a = reinterpret_cast<const uint32_t*>(word(e));
            r[2 * e] = e <= last ? __ldg(a) : 0;
            r[2 * e + 1] = e <= last ? __ldg(a + 1) : 0;
        }
    }
    return (uint32_t)(reinterpret_cast<uintptr_t>(first) & (N - 1));
}

template <class IN>
__device__ __forceinline__ void cut_item(Item<IN>& it, const uint32_t* r, uint32_t off, uint32_t P) {
    constexpr int W = Item<IN>::W;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t o = off == 8 ? 0 : (off + e * P * W) & (4 * W - 1);
        if constexpr (W == 2) {
            const bool high = o & 4;
            const uint32_t x = high ? r[4 * e + 1] : r[4 * e], y = high ? r[4 * e + 2] : r[4 * e + 1];
            const uint32_t z = high ? r[4 * e + 3] : r[4 * e + 2];
            it.w[2 * e] = __funnelshift_r(x, y, (o & 2) * 8);
            it.w[2 * e + 1] = __funnelshift_r(y, z, (o & 2) * 8);
        } else if constexpr (W == 1) {
            it.w[e] = __funnelshift_r(r[2 * e], r[2 * e + 1], o * 8);
        }
    }
}

// the four points' rows of one 16-byte column (8 channels) of an A piece
template <class T, class IN>
__device__ __forceinline__ void store_item(const Item<IN>& it, char* slot, int ch, int steps, int lane, bool vec) {
    constexpr int SPL = Form<T>::SPL;
    char* base = slot + (ch >> 1) * (16 * kAGroup) + (ch & 1) * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = neighbours<IN>(vec) ? 4 * lane + i : lane + 32 * i;
        uint32_t img[4][SPL];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(IN) == 4) {
                images<T>(make_float2(__uint_as_float(it.w[8 * e + i]), __uint_as_float(it.w[8 * e + 4 + i])), img[e]);
            } else if constexpr (sizeof(IN) == 2) {
                img[e][0] = __byte_perm(it.w[4 * e + i / 2], it.w[4 * e + 2 + i / 2], i & 1 ? 0x7632 : 0x5410);
            } else {
                const uint32_t two = __byte_perm(it.w[2 * e], it.w[2 * e + 1], (uint32_t)(i | (4 + i) << 4));
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffff), __NV_E4M3);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                images<T>(f, img[e]);  // exact
            }
        }
        char* at = base + (row >> 3) * kAGroup + (row & 7) * 16;
#pragma unroll
        for (int s = 0; s < SPL; ++s)
            *reinterpret_cast<uint4*>(at + s * steps * (16 * kAGroup)) =
                make_uint4(img[0][s], img[1][s], img[2][s], img[3][s]);
    }
}

// Two rows of 16-bit values, this thread's point in both (one word), as words of two points: of two neighbouring
// lanes the even one writes the first row and the odd one the second.
template <class T>
__device__ __forceinline__ void store_rows(T* at, uint32_t two, int lane, int left) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, two, 1);
    const bool odd = lane & 1;
    const uint32_t word = odd ? __byte_perm(other, two, 0x7632) : __byte_perm(two, other, 0x5410);
    if (left > (odd ? 1 : 0)) *reinterpret_cast<uint32_t*>(at + (odd ? TP - 1 : 0)) = word;
}

// the same rows in fp32
__device__ __forceinline__ void store_wide(float* at, float2 v, int left) {
    if (left > 0) at[0] = v.x;
    if (left > 1) at[TP] = v.y;
}

// an item of a 16-bit field as rows of 128 points in fp32
template <class T>
__device__ __forceinline__ void copy_wide(const Item<T>& it, float* __restrict__ z, int c0, int rows, int lane) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (c0 + e >= rows) break;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t h = (uint16_t)(it.w[2 * e + i / 2] >> (16 * (i & 1)));
                v[i] = to_f(*reinterpret_cast<const T*>(&h));
            }
            *reinterpret_cast<float4*>(z + (c0 + e) * TP + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

// the item's channels below `rows` as rows of 128 points
template <class T>
__device__ __forceinline__ void copy_item(const Item<T>& it, T* __restrict__ z, int c0, int rows, int lane, bool vec) {
    constexpr int W = Item<T>::W;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (c0 + e >= rows) break;
        T* to = z + (c0 + e) * TP;
        if (neighbours<T>(vec)) {
            if constexpr (W == 4)
                *reinterpret_cast<uint4*>(to + 4 * lane) =
                    make_uint4(it.w[4 * e], it.w[4 * e + 1], it.w[4 * e + 2], it.w[4 * e + 3]);
            else
                *reinterpret_cast<uint2*>(to + 4 * lane) = make_uint2(it.w[2 * e], it.w[2 * e + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (W == 4) to[lane + 32 * i] = __uint_as_float(it.w[4 * e + i]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// the block kernel
// ------------------------------------------------------------------------------------------------
// barriers, by index into the barrier area
struct Bars {
    uint64_t full_a[kMaxA], empty_a[kMaxA], full_b[kMaxB], empty_b[kMaxB];
    uint64_t d1[3], mid[3], g2[3], d2[2], d2_free[2], drain;
    uint32_t tmem;
    int abort_flag;
};

template <class T, class IN, bool BWD, bool GELU>
__global__ void __launch_bounds__(kThreads, 1)
k_block(const __grid_constant__ Params p, int* __restrict__ status) {
    constexpr int SPL = Form<T>::SPL, KC = Form<T>::KC, NP = Passes<SPL>::N, MID = Mid<T>::N;
    constexpr bool WIDE = sizeof(typename Scratch<T>::type) > sizeof(T);  // an fp32 scratch of a 16-bit field
    extern __shared__ __align__(1024) char sm[];
    const Plan& pl = p.pl;
    Bars& bar = *reinterpret_cast<Bars*>(sm + pl.o_bar);
    volatile int* abort_flag = &bar.abort_flag;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int i = 0; i < kMaxA; ++i) {
            tc::mbar_init(&bar.full_a[i], kProd);
            tc::mbar_init(&bar.empty_a[i], 1);
        }
        for (int i = 0; i < kMaxB; ++i) {
            tc::mbar_init(&bar.full_b[i], 1);
            tc::mbar_init(&bar.empty_b[i], 1);
        }
        for (int i = 0; i < 3; ++i) {
            tc::mbar_init(&bar.d1[i], 1);
            tc::mbar_init(&bar.mid[i], kEpi);
            tc::mbar_init(&bar.g2[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&bar.d2[i], 1);
            tc::mbar_init(&bar.d2_free[i], kEpi);
        }
        tc::mbar_init(&bar.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        bar.abort_flag = 0;
    }
    const float* vec = p.bias;
    if (pl.vec_smem) {  // k_pack's values, read by every middle: out of L2 they cost it 600 cycles a time
        float* v = reinterpret_cast<float*>(sm + pl.o_vec);
        for (int i = tid; i < 2 * pl.NH * pl.nJ + pl.N2; i += kThreads) v[i] = __ldg(p.bias + i);
        vec = v;
    }
    const float *bias_g = vec, *bias_u = vec + pl.NH * pl.nJ, *bias_2 = vec + 2 * pl.NH * pl.nJ;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(&bar.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bar.tmem, 0);
    auto give_up = [&]() {
        *abort_flag = 1;
        atomicExch(status, tc::kStatusMmaTimeout);
    };
    auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
        if (wait_for(b, parity, abort_flag)) return true;
        give_up();
        return false;
    };

    const int my = p.tiles > (int)blockIdx.x ? (p.tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    const int jobs = my * pl.nJ;
    const int nA = pl.nKx + pl.nKy;                       // A pieces of a job
    const int d1w = (BWD ? 3 : 2) * pl.NH;                // columns of a D1 buffer
    const int d2w = pl.N2 * (SPL == 3 ? 2 : 1);           // columns of a D2 buffer (D2c after D2)
    const uint32_t d2_0 = tmem + pl.n_d1 * d1w;
    const int lead = pl.n_d1 - 1;                         // first products run so many jobs ahead of second ones
    // D2 buffer of this CTA's run q, and how often it was used before
    auto d2_buf = [&](int q) { return pl.n_d2 == 2 ? q & 1 : 0; };
    auto d2_use = [&](int q) { return pl.n_d2 == 2 ? q >> 1 : q; };
    auto tile_at = [&](int k) { return (uint32_t)(p.tile0 + (int)blockIdx.x + k * (int)gridDim.x); };

    if (warp >= kEpi && warp < kMma) {
        // ------------------------------ x / e -> shared memory ------------------------------
        // a warp takes the 16-byte columns w, w + 4 of every piece; x and e have the same type in the backward
        const int w = warp - kEpi;
        constexpr int NI = KC / 32;                       // items a thread has in a piece
        // The place in the sequence of pieces (tile k, chunk j, piece kc), for the loads and for the stores,
        // which run one piece behind; the slot and its phase go with the stores.
        struct Place {
            int k, j, kc, i;
        };
        // What is in flight: a thread's part of a piece -- or, of a 16-bit field that is not aligned, of one item of it
        // (the words around its values are twice as many).
        struct Flight {
            uint32_t r[32], off[2];
        };
        constexpr int W = Item<IN>::W;
        const bool around = W < 4 && !p.vec;
        const int units = W == 2 && around ? NI : 1;
        const int chunks = pl.reuse ? 1 : pl.nJ;
        auto advance = [&](Place& q) {
            if (++q.i < units) return;
            q.i = 0;
            if (++q.kc < nA) return;
            q.kc = 0;
            if (++q.j == chunks) {
                q.j = 0;
                ++q.k;
            }
        };
        auto load = [&](Flight& f, Place& q) {
            if (q.k >= my) return;
            const bool is_x = !BWD || q.kc < pl.nKx;
            const IN* src = static_cast<const IN*>(is_x ? p.x : p.gy);
            const int k0 = (is_x ? q.kc : q.kc - pl.nKx) * KC;
            const int rows = is_x ? pl.C : pl.O;
            const uint32_t n0 = tile_at(q.k) * TP;
            if constexpr (W == 2) {
                if (around) {
                    f.off[0] = load_around<IN>(f.r, src, rows, k0 + (w + 4 * q.i) * 8, n0, lane, p);
                    advance(q);
                    return;
                }
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                if (W == 1 && around) f.off[i] = load_around<IN>(f.r + 16 * i, src, rows, k0 + (w + 4 * i) * 8, n0, lane, p);
                else load_item<IN>(f.r + (32 / NI) * i, src, rows, k0 + (w + 4 * i) * 8, n0, lane, p);
            }
            advance(q);
        };
        int slot = 0;
        uint32_t phase = 1;       // of the slot's last release: none is needed the first time
        auto put = [&](const Flight& f, Place& q) -> bool {
            if (q.k >= my) return false;
            const bool is_x = !BWD || q.kc < pl.nKx;
            const int pw = is_x ? piece_k(pl.Kx, KC, q.kc) : piece_k(pl.Ky, KC, q.kc - pl.nKx);
            if (q.i == 0 && !wait(&bar.empty_a[slot], phase)) return false;  // (true of a new barrier's phase 1)
            char* s = sm + pl.o_a + slot * pl.a_slot;
            // x and e go to the scratch too, once a tile
            const int results = 3 * Scratch<T>::PARTS * pl.H;
            const bool keep = BWD && p.z && p.z_rows > results && q.j == 0;
            const int c0 = (is_x ? q.kc : q.kc - pl.nKx) * KC;
            auto one = [&](const Item<IN>& it, int i) {
                const int ch = w + 4 * i;
                if (ch * 8 < pw) store_item<T, IN>(it, s, ch, pw / 16, lane, p.vec);
                if constexpr (BWD) {
                    const int64_t to =
                        ((int64_t)(tile_at(q.k) - p.tile0) * p.z_rows + results + (is_x ? 0 : pl.C)) * TP;
                    if (keep && WIDE)
                        copy_wide<T>(it, static_cast<float*>(p.z) + to, c0 + ch * 8, is_x ? pl.C : pl.O, lane);
                    else if (keep)
                        copy_item<T>(it, static_cast<T*>(p.z) + to, c0 + ch * 8, is_x ? pl.C : pl.O, lane, p.vec);
                }
            };
            Item<IN> it;
            bool single = false;
            if constexpr (W == 2) {
                if (around) {
                    single = true;
                    cut_item<IN>(it, f.r, f.off[0], p.P);
                    one(it, q.i);
                }
            }
            if (!single) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (W == 1 && around) {
                        cut_item<IN>(it, f.r + 16 * i, f.off[i], p.P);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8 * W; ++e) it.w[e] = f.r[(32 / NI) * i + e];
                    }
                    one(it, i);
                }
            }
            if (q.i == units - 1) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bar.full_a[slot]);
                if (++slot == pl.na) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            advance(q);
            return true;
        };
        // the next piece is in flight while this one waits for its slot and is written
        Flight c, d;
        Place in{0, 0, 0, 0}, at = in;
        load(c, in);
        while (true) {
            load(d, in);
            if (!put(c, at)) break;
            load(c, in);
            if (!put(d, at)) break;
        }
    } else if (warp == kLoad) {
        // ------------------------------ weights -> shared memory ------------------------------
        if (lane == 0 && jobs > 0) {
            const uint32_t sb = tc::smem_u32(sm + pl.o_b);
            if (pl.resident) {
                bulk_copy(sb, p.packed, (uint32_t)(pl.nJ * pl.job_bytes), &bar.full_b[0]);
                tc::mbar_wait(&bar.full_b[0], 0, nullptr);  // no copy outlives the CTA (bounded)
            } else {
                int q = 0;
                bool ok = true;
                auto push = [&](const char* src, int rows, int pw) -> int {
                    const int slot = q % pl.nb, use = q / pl.nb, bytes = rows * pw * 2 * SPL;
                    if (use > 0 && !wait(&bar.empty_b[slot], (uint32_t)(use - 1) & 1)) {
                        ok = false;
                        return 0;
                    }
                    bulk_copy(sb + slot * pl.b_slot, src, (uint32_t)bytes, &bar.full_b[slot]);
                    ++q;
                    return bytes;
                };
                for (int J = 0; J < jobs + lead && ok; ++J) {  // in the order of the MMA warp
                    if (J < jobs) {
                        const char* src = p.packed + (int64_t)(J % pl.nJ) * pl.job_bytes;
                        for (int kc = 0; kc < pl.nKx && ok; ++kc) src += push(src, 2 * pl.NH, piece_k(pl.Kx, KC, kc));
                        for (int kc = 0; kc < pl.nKy && ok; ++kc) src += push(src, pl.NH, piece_k(pl.Ky, KC, kc));
                    }
                    if (J >= lead && ok) {
                        const char* src = p.packed + (int64_t)((J - lead) % pl.nJ) * pl.job_bytes +
                                          (int64_t)pl.NH * (2 * pl.Kx + pl.Ky) * 2 * SPL;
                        for (int m = 0; m < (BWD ? 2 : 1); ++m)
                            for (int kc = 0; kc < pl.nH && ok; ++kc) src += push(src, pl.N2, piece_k(pl.NH, KC, kc));
                    }
                }
                for (int i = 0; i < pl.nb && i < q; ++i) {  // no copy outlives the CTA (bounded)
                    const int last = q - 1 - i;
                    tc::mbar_wait(&bar.full_b[last % pl.nb], (uint32_t)(last / pl.nb) & 1, nullptr);
                }
            }
        }
    } else if (warp == kMma) {
        // ------------------------------ MMA issue ------------------------------
        if (jobs > 0) {
            const uint32_t leader = elect_one();
            const uint32_t sa = tc::smem_u32(sm + pl.o_a), sb = tc::smem_u32(sm + pl.o_b);
            constexpr uint32_t fmt = Form<T>::kFmt;
            const uint32_t id_g = idesc_of(fmt, 2 * pl.NH), id_f = idesc_of(fmt, pl.NH), id_2 = idesc_of(fmt, pl.N2);
            auto all = [&](uint64_t* b, uint32_t parity) -> bool {  // the warp stays together
                return __all_sync(0xffffffffu, wait(b, parity));
            };
            int qs = 0, a0 = 0;            // weight slot; slot of the job's (reuse: the tile's) first A piece
            uint32_t qp = 0, ap = 0;       // their phases
            bool ok = !pl.resident || all(&bar.full_b[0], 0);
            // the images of the next weight piece (`at`: its place among all of them, when resident)
            auto weights = [&](int at) -> uint32_t {
                if (pl.resident) return sb + (uint32_t)at;
                if (!all(&bar.full_b[qs], qp)) ok = false;
                return sb + (uint32_t)(qs * pl.b_slot);
            };
            auto weights_done = [&]() {
                if (pl.resident) return;
                commit(&bar.empty_b[qs], leader);
                if (++qs == pl.nb) {
                    qs = 0;
                    qp ^= 1;
                }
            };
            // D (columns d ..) (+)= A piece from shared memory x B piece of N rows; the smaller products first
            auto product_ss = [&](uint32_t d, uint32_t at, uint32_t bt, uint32_t id, int N, int pw, bool acc) {
                const int steps = pw / 16;
                uint64_t da[SPL], db[SPL];
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    da[s] = desc_of(at + s * steps * (16 * kAGroup), kAGroup);
                    db[s] = desc_of(bt + s * N * pw * 2, 256);
                }
                const uint32_t bstep = N * 2;
                if constexpr (NP > 1) {
#pragma unroll
                    for (int ks = 0; ks < KC / 16; ++ks) {
                        if (ks >= steps) break;
#pragma unroll
                        for (int i = 1; i < NP; ++i)
                            mma_ss(d, da[Passes<SPL>::a(i)] + ks * kAGroup, db[Passes<SPL>::b(i)] + ks * bstep, id,
                                   acc || ks > 0 || i > 1, leader);
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KC / 16; ++ks) {
                    if (ks >= steps) break;
                    mma_ss(d, da[0] + ks * kAGroup, db[0] + ks * bstep, id, NP > 1 || acc || ks > 0, leader);
                }
            };
            // ... x A images in tensor memory; image s of the K step of hidden group g at column col[s] + 16 g; the
            // smaller products in the N columns after D's
            auto product_ts = [&](uint32_t d, const uint32_t (&col)[MID], uint32_t bt, int N, int pw, bool acc, int g0) {
                uint64_t db[SPL];
#pragma unroll
                for (int s = 0; s < SPL; ++s) db[s] = desc_of(bt + s * N * pw * 2, 256);
                const uint32_t bstep = N * 2;
#pragma unroll
                for (int ks = 0; ks < KC / 16; ++ks) {
                    if (ks >= pw / 16) break;
#pragma unroll
                    for (int i = 0; i < (SPL == 1 ? MID : NP); ++i) {
                        if constexpr (SPL == 1)
                            mma_ts(d, col[i] + 16 * (g0 + ks), db[0] + ks * bstep, id_2, i > 0 || acc || ks > 0, leader);
                        else
                            mma_ts(i ? d + N : d, col[Passes<SPL>::a(i)] + 16 * (g0 + ks),
                                   db[Passes<SPL>::b(i)] + ks * bstep, id_2, i > 1 || acc || ks > 0, leader);
                    }
                }
            };
            int j1 = 0, j2 = 0;            // chunk of the first and of the second product
            int i2 = 0, q2 = 0;            // the second one's chunk of its run of D2, and the run
            int b1 = 0, b2 = 0;            // D1 buffers of the two
            uint32_t p1 = 1, p2 = 0;       // phases: of the first one's last second product, of the second one's middle
            for (int J = 0; J < jobs + lead && ok; ++J) {
                if (J < jobs) {  // first product of job J
                    if (!all(&bar.g2[b1], p1)) break;  // (true of a new barrier's phase 1)
                    fence_after();
                    const uint32_t d = tmem + b1 * d1w;
                    const bool last = j1 == pl.nJ - 1;
                    int at = j1 * pl.job_bytes, slot = a0;
                    uint32_t phase = ap;
                    for (int kc = 0; kc < nA; ++kc) {
                        const bool is_x = kc < pl.nKx;
                        const int pw = is_x ? piece_k(pl.Kx, KC, kc) : piece_k(pl.Ky, KC, kc - pl.nKx);
                        const int N = is_x ? 2 * pl.NH : pl.NH;
                        if (!all(&bar.full_a[slot], phase)) ok = false;
                        const uint32_t wb = weights(at);
                        if (!ok) break;
                        fence_after();
                        product_ss(is_x ? d : d + 2 * pl.NH, sa + slot * pl.a_slot, wb, is_x ? id_g : id_f, N, pw,
                                   kc != 0 && kc != pl.nKx);
                        at += N * pw * 2 * SPL;
                        weights_done();
                        if (!pl.reuse || last) commit(&bar.empty_a[slot], leader);
                        if (++slot == pl.na) {
                            slot = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    commit(&bar.d1[b1], leader);
                    if (++b1 == pl.n_d1) {
                        b1 = 0;
                        p1 ^= 1;
                    }
                    if (!pl.reuse || last) {
                        a0 = slot;
                        ap = phase;
                    }
                    j1 = last ? 0 : j1 + 1;
                }
                if (J >= lead) {  // second product of job J - lead
                    if (!all(&bar.mid[b2], p2)) break;
                    const int e = d2_buf(q2);
                    if (i2 == 0 && d2_use(q2) > 0 && !all(&bar.d2_free[e], (uint32_t)(d2_use(q2) - 1) & 1)) break;
                    const uint32_t d2 = d2_0 + e * d2w;
                    fence_after();
                    const uint32_t d = tmem + b2 * d1w;
                    int at = j2 * pl.job_bytes + pl.NH * (2 * pl.Kx + pl.Ky) * 2 * SPL;
#pragma unroll
                    for (int m = 0; m < (BWD ? 2 : 1); ++m) {
                        uint32_t col[MID];  // the places that the middle gave the images
                        if constexpr (SPL == 1) {
                            col[0] = d + m * pl.NH;
                            col[1] = col[0] + 8;
                        } else {
                            col[0] = m ? d + pl.NH + 8 : d;
                            col[1] = m ? d + 2 * pl.NH : d + 8;
                            col[2] = m ? d + 2 * pl.NH + 8 : d + pl.NH;
                        }
                        for (int kc = 0; kc < pl.nH && ok; ++kc) {
                            const int pw = piece_k(pl.NH, KC, kc);
                            const uint32_t wb = weights(at);
                            if (!ok) break;
                            fence_after();
                            product_ts(d2, col, wb, pl.N2, pw, i2 != 0 || m != 0 || kc != 0, kc * (KC / 16));
                            at += pl.N2 * pw * 2 * SPL;
                            weights_done();
                        }
                    }
                    if (!ok) break;
                    commit(&bar.g2[b2], leader);
                    if (++b2 == pl.n_d1) {
                        b2 = 0;
                        p2 ^= 1;
                    }
                    if (++j2 == pl.nJ) j2 = 0;
                    if (++i2 == pl.per || j2 == 0) {
                        commit(&bar.d2[e], leader);
                        i2 = 0;
                        ++q2;
                    }
                }
            }
            // every MMA issued has completed before the tensor memory is freed (bounded)
            commit(&bar.drain, leader);
            tc::mbar_wait(&bar.drain, 0, nullptr);
        }
    } else if (warp < kEpi) {
        // ------------------------------ middle ------------------------------
        const int quad = warp & 3, part = warp >> 2;      // lane quadrant; which 16-column groups
        const int row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const int groups = pl.NH / 16;

        int b = 0;                 // D1 buffer and its phase
        uint32_t phase = 0;
        auto middle = [&](int k, int j) -> bool {
            const uint32_t tile = tile_at(k), n = tile * TP + row;
            const bool valid = n < p.points;
            float sc = 1.f;
            if constexpr (sizeof(IN) == 1) sc = valid ? __ldg(p.scale + n) : 0.f;
            if (!wait(&bar.d1[b], phase)) return false;
            fence_after();
            const uint32_t d = tmem + b * d1w + lanes;
            for (int g = part; g < groups; g += kEpi / 4) {
                float vg[16], vu[16];
                ld16(d + 16 * g, vg);
                ld16(d + pl.NH + 16 * g, vu);
                const int h0 = j * pl.NH + 16 * g;
                float4 bg[4], bu[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bg[i] = reinterpret_cast<const float4*>(bias_g + h0)[i];
                    bu[i] = reinterpret_cast<const float4*>(bias_u + h0)[i];
                }
                wait_ld(vg);
                wait_ld(vu);
                float2 g2[8], u2[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 a = bg[i], c = bu[i];
                    g2[2 * i] = __ffma2_rn(make_float2(vg[4 * i], vg[4 * i + 1]), both(sc), make_float2(a.x, a.y));
                    g2[2 * i + 1] = __ffma2_rn(make_float2(vg[4 * i + 2], vg[4 * i + 3]), both(sc), make_float2(a.z, a.w));
                    u2[2 * i] = __ffma2_rn(make_float2(vu[4 * i], vu[4 * i + 1]), both(sc), make_float2(c.x, c.y));
                    u2[2 * i + 1] = __ffma2_rn(make_float2(vu[4 * i + 2], vu[4 * i + 3]), both(sc), make_float2(c.z, c.w));
                }
                if constexpr (!BWD) {
                    uint32_t w[MID][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float2 slope;
                        uint32_t t[MID];
                        mid_images<T>(__fmul2_rn(activation<GELU>(g2[i], slope), u2[i]), t);
#pragma unroll
                        for (int s = 0; s < MID; ++s) w[s][i] = t[s];
                    }
                    st8(d + 16 * g, w[0]);
                    st8(d + 16 * g + 8, w[1]);
                    if constexpr (SPL == 3) st8(d + pl.NH + 16 * g, w[MID - 1]);
                } else {
                    float vf[16];
                    ld16(d + 2 * pl.NH + 16 * g, vf);
                    wait_ld(vf);
                    const int64_t z_at = ((int64_t)(tile - p.tile0) * p.z_rows + h0) * TP + row;
                    T* z = static_cast<T*>(p.z) + z_at;
                    float* zw = static_cast<float*>(p.z) + z_at;
                    T *zu = z + pl.H * TP, *zh = zu + pl.H * TP;
                    const int left = p.z ? pl.H - h0 : 0;
                    uint32_t w[2][MID][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float2 slope;
                        const float2 a = activation<GELU>(g2[i], slope);
                        // points past the last one are zeros in the scratch
                        const float2 f = valid ? make_float2(vf[2 * i], vf[2 * i + 1]) : both(0.f);
                        const float2 h = valid ? __fmul2_rn(a, u2[i]) : both(0.f);
                        const float2 dg = __fmul2_rn(__fmul2_rn(f, u2[i]), slope), du = __fmul2_rn(f, a);
                        uint32_t t[MID], r[MID];
                        mid_images<T>(dg, t);
                        mid_images<T>(du, r);
#pragma unroll
                        for (int s = 0; s < MID; ++s) {
                            w[0][s][i] = t[s];
                            w[1][s][i] = r[s];
                        }
                        if constexpr (WIDE) {
                            store_wide(zw + 2 * i * TP, dg, left - 2 * i);
                            store_wide(zw + (pl.H + 2 * i) * TP, du, left - 2 * i);
                            store_wide(zw + (2 * pl.H + 2 * i) * TP, h, left - 2 * i);
                        } else if constexpr (SPL == 1) {
                            uint32_t o[MID];
                            mid_images<T>(h, o);
#pragma unroll
                            for (int s = 0; s < MID; ++s) {
                                const int at = (3 * s * pl.H + 2 * i) * TP;
                                store_rows(z + at, t[s], lane, left - 2 * i);
                                store_rows(zu + at, r[s], lane, left - 2 * i);
                                store_rows(zh + at, o[s], lane, left - 2 * i);
                            }
                        } else {
                            if (2 * i < left) {
                                z[2 * i * TP] = dg.x;
                                zu[2 * i * TP] = du.x;
                                zh[2 * i * TP] = h.x;
                            }
                            if (2 * i + 1 < left) {
                                z[(2 * i + 1) * TP] = dg.y;
                                zu[(2 * i + 1) * TP] = du.y;
                                zh[(2 * i + 1) * TP] = h.y;
                            }
                        }
                    }
                    if constexpr (SPL == 1) {
                        st8(d + 16 * g, w[0][0]);
                        st8(d + 16 * g + 8, w[0][1]);
                        st8(d + pl.NH + 16 * g, w[1][0]);
                        st8(d + pl.NH + 16 * g + 8, w[1][1]);
                    } else {
                        st8(d + 16 * g, w[0][0]);
                        st8(d + 16 * g + 8, w[0][1]);
                        st8(d + pl.NH + 16 * g, w[0][2]);
                        st8(d + pl.NH + 16 * g + 8, w[1][0]);
                        st8(d + 2 * pl.NH + 16 * g, w[1][1]);
                        st8(d + 2 * pl.NH + 16 * g + 8, w[1][2]);
                    }
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bar.mid[b]);
            if (++b == pl.n_d1) {
                b = 0;
                phase ^= 1;
            }
            return true;
        };
        // run r of tile k, the CTA's run q
        auto output = [&](int k, int r, int q) -> bool {
            const uint32_t n = tile_at(k) * TP + row;
            const bool valid = n < p.points;
            const int width = BWD ? pl.C : pl.O;      // the field's channels
            const uint32_t b = valid ? sample_of(p, n) : 0;
            T* y = static_cast<T*>(p.out) + ((int64_t)b * width + pl.col0) * p.P + (valid ? n - b * p.P : 0);
            const int e = d2_buf(q);
            if (!wait(&bar.d2[e], (uint32_t)d2_use(q) & 1)) return false;
            fence_after();
            const uint32_t d2 = d2_0 + e * d2w;
            const int n16 = pl.N2 / 16;
            if (part >= n16) {  // a warp without columns
                fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bar.d2_free[e]);
            }
            for (int g = part; g < n16; g += kEpi / 4) {
                float v[16];
                ld16(d2 + lanes + 16 * g, v);
                wait_ld(v);
                if constexpr (SPL == 3) {
                    float c[16];
                    ld16(d2 + pl.N2 + lanes + 16 * g, c);
                    wait_ld(c);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] += c[i];
                }
                if (g + kEpi / 4 >= n16) {  // read: the next second product may begin while this goes out
                    fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&bar.d2_free[e]);
                }
                if (!BWD && r == pl.runs - 1) {  // all loads before the stores, which might alias them for all the compiler knows
                    const float4* b2 = reinterpret_cast<const float4*>(bias_2 + 16 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 c = b2[i];
                        v[4 * i] += c.x;
                        v[4 * i + 1] += c.y;
                        v[4 * i + 2] += c.z;
                        v[4 * i + 3] += c.w;
                    }
                }
                if (!valid || !p.out) continue;
                T* yg = y + (int64_t)(16 * g) * p.P;
                const int left = pl.cols - 16 * g;
                if constexpr (SPL == 3) {
                    if (r > 0) {  // the runs before this one, which this thread has written
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (i < left) v[i] += to_f(yg[(int64_t)i * p.P]);
                    }
                }
                if (left >= 16) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) yg[(int64_t)i * p.P] = from_f<T>(v[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (i < left) yg[(int64_t)i * p.P] = from_f<T>(v[i]);
                }
            }
            return true;
        };
        // a run goes out after the next one's first middle
        bool ok = true;
        int q = 0, k0 = 0, r0 = 0;  // runs begun; tile and place in it of the last one
        for (int k = 0; k < my && ok; ++k) {
            for (int j = 0, i = 0, r = 0; j < pl.nJ && ok; ++j) {
                ok = middle(k, j);
                if (i == 0) {
                    if (ok && q > 0) ok = output(k0, r0, q - 1);
                    ++q;
                    k0 = k;
                    r0 = r;
                }
                if (++i == pl.per) {
                    i = 0;
                    ++r;
                }
            }
        }
        if (ok && my > 0) output(k0, r0, q - 1);
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------------------------------------------
// weight gradients
// ------------------------------------------------------------------------------------------------
constexpr int kPromote = 8;                   // pieces an accumulator runs before it goes to registers
constexpr int kImages = 2;                    // fp32: stages of split operands

// A piece is 128 bytes of points of up to 128 rows of each operand, as a 128-byte-swizzled tensor copy leaves them:
// for bf16 that is the MMA's own K-major layout and the pieces are multiplied as they land, both parts of A with B.
template <class T> struct WForm {
    // warps 0..7: accumulators; then fp32 splitting (four warps an operand) and row sums, MMA issue, copies
    static constexpr int WORK = sizeof(T) == 4 ? 8 : 4, MMA = 8 + WORK, LOAD = MMA + 1, THREADS = 32 * (LOAD + 1);
    static constexpr int KC = 128 / (int)sizeof(T);
    static constexpr int STAGES = sizeof(T) == 4 ? 3 : 4;
    static constexpr int PARTS = Scratch<T>::PARTS;
    static constexpr int ONE = 128 * 128;                            // bytes of one operand's rows
    static constexpr int RAW = (1 + PARTS) * ONE;                    // A rows, then B rows, then A's second part
    static constexpr int IMG = sizeof(T) == 4 ? 128 * KC * 2 : 0;    // one image of one operand
    static constexpr int SPLIT = 2 * Form<T>::SPL * IMG;
    static constexpr int BODY = STAGES * RAW + (sizeof(T) == 4 ? kImages * SPLIT : 0);
};

struct WParams {
    float* partial;            // [split][tile][128][128]
    double* sums;              // [split][2 H + O] row sums of dg, du and e (may be NULL)
    int C, H, O;
    int rows;                  // rows of a tile of the scratch (3 H PARTS are dg, du and h)
    int tile0, per_sample;     // x and e in place: the slab's first tile, tiles of a sample; per_sample 0: in the scratch
    int pieces;                // pieces of KC points in the slab
    int splits;
    int nC, nO;                // column tiles of x and of e
    int mX, mH;                // row tiles of [dg; du] and of h
    int accumulate;            // add to the partial sums of the slabs before
};

struct WBars {
    uint64_t raw[6], raw_free[6], img[kImages], img_free[kImages], acc[2], acc_free[2], drain;
    uint32_t tmem;
    int abort_flag;
};

__device__ __forceinline__ uint64_t desc_128b(uint32_t addr) {  // K-major rows of 128 bytes, 128-byte swizzle
    return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// CTA = (tile, split).  Tile: 128 rows of the scratch (rows of [dg; du] against rows of x, rows of h against rows of
// e) x up to 128 columns; K: the split's share of the slab's points.
template <class T>
__global__ void __launch_bounds__(WForm<T>::THREADS, 1)
k_wgrad(const __grid_constant__ CUtensorMap mg, const __grid_constant__ CUtensorMap mh,
        const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap me, const __grid_constant__ WParams p, int* __restrict__ status) {
    using W = WForm<T>;
    constexpr int SPL = Form<T>::SPL, KC = W::KC, NP = Passes<SPL>::N, S = W::STAGES;
    constexpr bool kSplit = SPL > 1;
    constexpr int DW = kSplit ? 256 : 128;      // columns of an accumulator (and the smaller products')
    extern __shared__ __align__(1024) char sm[];
    WBars& bar = *reinterpret_cast<WBars*>(sm + W::BODY);
    volatile int* abort_flag = &bar.abort_flag;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int tiles = p.mX * p.nC + p.mH * p.nO;
    const int tile = (int)blockIdx.x % tiles, split = (int)blockIdx.x / tiles;
    const bool of_x = tile < p.mX * p.nC;
    const int mt = of_x ? tile / p.nC : (tile - p.mX * p.nC) / p.nO, nt = of_x ? tile % p.nC : (tile - p.mX * p.nC) % p.nO;
    const int a_rows = (of_x ? 2 * p.H : p.H) - mt * 128;    // rows left from the tile's first
    const int b_rows = (of_x ? p.C : p.O) - nt * 128;
    const int n = imin(128, up16(b_rows));
    const int k0 = (int)((int64_t)p.pieces * split / p.splits), k1 = (int)((int64_t)p.pieces * (split + 1) / p.splits);
    const int steps = k1 - k0, runs = (steps + kPromote - 1) / kPromote;
    const bool want_a = p.sums && of_x && nt == 0, want_b = p.sums && !of_x && mt == 0;
    const bool working = kSplit || want_a || want_b;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            tc::mbar_init(&bar.raw[i], 1);
            tc::mbar_init(&bar.raw_free[i], kSplit ? W::WORK : working ? W::WORK + 1 : 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&bar.img[i], W::WORK);
            tc::mbar_init(&bar.img_free[i], 1);
            tc::mbar_init(&bar.acc[i], 1);
            tc::mbar_init(&bar.acc_free[i], 8);
        }
        tc::mbar_init(&bar.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        bar.abort_flag = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&bar.tmem)),
                     "n"(2 * DW)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bar.tmem, 0);
    auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
        if (wait_for(b, parity, abort_flag)) return true;
        *abort_flag = 1;
        atomicExch(status, tc::kStatusMmaTimeout);
        return false;
    };
    char* split_at = sm + S * W::RAW;

    if (warp == W::LOAD) {
        // ------------------------------ scratch -> shared memory ------------------------------
        if (lane == 0) {
            const CUtensorMap* mb = of_x ? &mx : &me;
            const int a0 = (of_x ? 0 : 2 * p.H) + mt * 128;
            const int b0 = nt * 128 + (p.per_sample ? 0 : 3 * W::PARTS * p.H + (of_x ? 0 : p.C));
            const CUtensorMap* ma = of_x ? &mg : &mh;
            const uint32_t bytes =
                (uint32_t)(W::PARTS * imin(128, of_x ? 2 * p.H : p.H) + imin(128, of_x ? p.C : p.O)) * 128;
            int k = 0;
            for (; k < steps; ++k) {
                const int slot = k % S, use = k / S;
                if (use > 0 && !wait(&bar.raw_free[slot], (uint32_t)(use - 1) & 1)) break;
                const int at = (k0 + k) * KC, t = at / TP, c = at % TP;
                const uint32_t dst = tc::smem_u32(sm + slot * W::RAW);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(&bar.raw[slot])),
                             "r"(bytes)
                             : "memory");
                auto copy = [&](uint32_t to, const CUtensorMap* m, int c, int row) {
                    asm volatile(
                        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
                        "%3}], [%4];" ::"r"(to),
                        "l"(reinterpret_cast<uint64_t>(m)), "r"(c), "r"(row), "r"(tc::smem_u32(&bar.raw[slot]))
                        : "memory");
                };
                copy(dst, ma, c, t * p.rows + a0);
                if (W::PARTS > 1) copy(dst + 2 * W::ONE, ma, c, t * p.rows + 3 * p.H + a0);
                if (p.per_sample) {
                    const int s = (p.tile0 + t) / p.per_sample, first = (p.tile0 + t - s * p.per_sample) * TP;
                    copy(dst + W::ONE, mb, first + c, s * (of_x ? p.C : p.O) + b0);
                } else {
                    copy(dst + W::ONE, mb, c, t * p.rows + b0);
                }
            }
            for (int i = 0; i < S && i < k; ++i)  // no copy outlives the CTA (bounded)
                tc::mbar_wait(&bar.raw[(k - 1 - i) % S], (uint32_t)((k - 1 - i) / S) & 1, nullptr);
        }
    } else if (warp >= 8 && warp < W::MMA) {
        // ------------------------------ splitting and row sums: a thread has a row of each operand ----------------
        const int r = (tid - 256) & 127, o = kSplit ? (tid - 256) >> 7 : want_b;  // row, operand
        const bool summing = o ? want_b : want_a;
        double sum = 0.0;
        auto row_of = [&](const char* raw, float (&v)[KC]) {
            const char* row = raw + r * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const uint4 q = *reinterpret_cast<const uint4*>(row + ((c ^ (r & 7)) * 16));
                const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
                for (int i = 0; i < KC / 8; ++i) v[c * (KC / 8) + i] = to_f(e[i]);
            }
        };
        auto add = [&](const float (&v)[KC]) {  // a piece's values in fp32, the pieces in 64 bits
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KC; ++i) s[i % 4] += v[i];
            sum += (double)((s[0] + s[1]) + (s[2] + s[3]));
        };
        for (int k = 0; working && k < steps; ++k) {
            const int slot = k % S;
            if (!wait(&bar.raw[slot], (uint32_t)(k / S) & 1)) break;
            const char* raw = sm + slot * W::RAW;
            float v[KC];
            if constexpr (kSplit) {
                const int si = k % kImages, use = k / kImages;
                if (use > 0 && !wait(&bar.img_free[si], (uint32_t)(use - 1) & 1)) break;
                if (!o || r < n) {
                    row_of(raw + o * W::ONE, v);
                    char* to = split_at + si * W::SPLIT + o * SPL * W::IMG + (r >> 3) * 256 + (r & 7) * 16;
#pragma unroll
                    for (int ch = 0; ch < KC / 8; ++ch) {
                        uint32_t img[4][SPL];
#pragma unroll
                        for (int e = 0; e < 4; ++e) images<T>(make_float2(v[8 * ch + 2 * e], v[8 * ch + 2 * e + 1]), img[e]);
#pragma unroll
                        for (int q = 0; q < SPL; ++q)
                            *reinterpret_cast<uint4*>(to + q * W::IMG + (ch >> 1) * (128 * 32) + (ch & 1) * 128) =
                                make_uint4(img[0][q], img[1][q], img[2][q], img[3][q]);
                    }
                    if (summing) add(v);
                }
            } else {
                row_of(raw + o * W::ONE, v);
                add(v);
                if (W::PARTS > 1 && !o) {
                    row_of(raw + 2 * W::ONE, v);
                    add(v);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (kSplit) tc::mbar_arrive(&bar.img[k % kImages]);
                tc::mbar_arrive(&bar.raw_free[slot]);
            }
        }
        if (summing && r < (o ? b_rows : a_rows)) {
            double* out = p.sums + (int64_t)split * (2 * p.H + p.O) + (o ? 2 * p.H + nt * 128 : mt * 128) + r;
            *out = p.accumulate ? *out + sum : sum;
        }
    } else if (warp == W::MMA) {
        // ------------------------------ MMA issue ------------------------------
        const uint32_t leader = elect_one();
        const uint32_t id = idesc_of(Form<T>::kFmt, n);
        auto all = [&](uint64_t* b, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(b, parity)); };
        constexpr int Q = kSplit ? kImages : S;
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int r = 0; r < runs && ok; ++r) {
            const int buf = r & 1;
            if (r >= 2 && !all(&bar.acc_free[buf], (uint32_t)((r >> 1) - 1) & 1)) break;
            fence_after();
            const int end = imin(steps, (r + 1) * kPromote);
            for (int k = r * kPromote; k < end; ++k) {
                if (!all(kSplit ? &bar.img[slot] : &bar.raw[slot], phase)) {
                    ok = false;
                    break;
                }
                fence_after();
                const bool first = k == r * kPromote;
                const uint32_t d = tmem + buf * DW;
                if constexpr (kSplit) {
                    const uint32_t at = tc::smem_u32(split_at + slot * W::SPLIT);
                    const uint64_t a0 = desc_of(at, 256), b0 = desc_of(at + SPL * W::IMG, 256);
#pragma unroll
                    for (int ks = 0; ks < KC / 16; ++ks) {
#pragma unroll
                        for (int i = 0; i < NP; ++i)
                            mma_ss(d + (i ? 128 : 0), a0 + (Passes<SPL>::a(i) * W::IMG + ks * 128 * 32) / 16,
                                   b0 + (Passes<SPL>::b(i) * W::IMG + ks * 128 * 32) / 16, id, i > 1 || ks > 0 || !first,
                                   leader);
                    }
                    commit(&bar.img_free[slot], leader);
                } else {
                    const uint32_t at = tc::smem_u32(sm + slot * W::RAW);
                    const uint64_t a0 = desc_128b(at), b0 = desc_128b(at + W::ONE), a1 = desc_128b(at + 2 * W::ONE);
#pragma unroll
                    for (int ks = 0; ks < KC / 16; ++ks) {
                        mma_ss(d, a0 + 2 * ks, b0 + 2 * ks, id, ks > 0 || !first, leader);
                        mma_ss(d, a1 + 2 * ks, b0 + 2 * ks, id, true, leader);
                    }
                    commit(&bar.raw_free[slot], leader);
                }
                if (++slot == Q) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (ok) commit(&bar.acc[buf], leader);
        }
        // every MMA issued has completed before the tensor memory is freed (bounded)
        commit(&bar.drain, leader);
        tc::mbar_wait(&bar.drain, 0, nullptr);
    } else {
        // ------------------------------ accumulators -> registers -> partial sums ------------------------------
        const int quad = warp & 3, half = warp >> 2, row = quad * 32 + lane;
        float sum[4][16];   // groups of 16 columns half, half + 2, ...
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[g][i] = 0.f;
        bool ok = true;
        for (int r = 0; r < runs; ++r) {
            const int buf = r & 1;
            if (!wait(&bar.acc[buf], (uint32_t)(r >> 1) & 1)) {
                ok = false;
                break;
            }
            fence_after();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if ((half + 2 * g) * 16 < n) {
                    const uint32_t at = tmem + buf * DW + (half + 2 * g) * 16 + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        float v[8], c[8] = {};
                        tc::tmem_ld8(at + i, v);
                        if (kSplit) tc::tmem_ld8(at + 128 + i, c);
                        asm volatile("tcgen05.wait::ld.sync.aligned;"
                                     : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                                       "+f"(v[7]), "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]), "+f"(c[4]), "+f"(c[5]),
                                       "+f"(c[6]), "+f"(c[7])
                                     :
                                     : "memory");
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum[g][i + e] += kSplit ? v[e] + c[e] : v[e];
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bar.acc_free[buf]);
        }
        if (ok && row < a_rows) {
            float* out = p.partial + ((int64_t)split * tiles + tile) * (128 * 128) + row * 128;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if ((half + 2 * g) * 16 >= n) continue;
                float4* o4 = reinterpret_cast<float4*>(out + (half + 2 * g) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 v = make_float4(sum[g][4 * i], sum[g][4 * i + 1], sum[g][4 * i + 2], sum[g][4 * i + 3]);
                    if (p.accumulate) {
                        const float4 o = o4[i];
                        v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
                    }
                    o4[i] = v;
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * DW));
}

// the splits' partial sums added in 64 bits, in order
template <class T>
__global__ void __launch_bounds__(128)
k_finish(WParams p, T* __restrict__ gwg, T* __restrict__ gwu, T* __restrict__ gwd, T* __restrict__ gbg,
         T* __restrict__ gbu, T* __restrict__ gbd) {
    const int tiles = p.mX * p.nC + p.mH * p.nO;
    const int rows = 3 * p.H, r = blockIdx.x;
    if (r < rows) {
        const bool of_x = r < 2 * p.H;
        const int q = of_x ? r : r - 2 * p.H, cols = of_x ? p.C : p.O;
        for (int c = threadIdx.x; c < cols; c += 128) {
            const int tile = of_x ? q / 128 * p.nC + c / 128 : p.mX * p.nC + q / 128 * p.nO + c / 128;
            const float* src = p.partial + (int64_t)tile * (128 * 128) + q % 128 * 128 + c % 128;
            double s = 0.0;
            for (int k = 0; k < p.splits; ++k) s += (double)src[(int64_t)k * tiles * (128 * 128)];
            if (r < p.H) {
                if (gwg) gwg[(int64_t)r * p.C + c] = from_f<T>((float)s);
            } else if (of_x) {
                if (gwu) gwu[(int64_t)(r - p.H) * p.C + c] = from_f<T>((float)s);
            } else if (gwd) {
                gwd[(int64_t)c * p.H + q] = from_f<T>((float)s);
            }
        }
        return;
    }
    const int all = 2 * p.H + p.O;
    for (int c = (r - rows) * 128 + threadIdx.x; c < all; c += (gridDim.x - rows) * 128) {
        T* out = c < p.H ? gbg : c < 2 * p.H ? gbu : gbd;
        if (!out) continue;
        double s = 0.0;
        for (int k = 0; k < p.splits; ++k) s += p.sums[(int64_t)k * all + c];
        out[c < p.H ? c : c < 2 * p.H ? c - p.H : c - 2 * p.H] = from_f<T>((float)s);
    }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
// How a call is cut.  An fp32 launch takes at most 128 output channels (D2 and D2c); more are several launches, each
// with the whole first product.  Tensor memory: two D1 buffers and D2 (fp32: and D2c) in 512 columns, so the
// backward's chunk (three columns a hidden channel) is 64 wide when D2 takes up to 128 of them and 32 above; what is
// left holds a third D1, or a second D2, or both.  Shared memory: the weights stay when they
// leave room for two pieces of A, otherwise two to six pieces of each stream.
template <class T>
bool make_plan(const nop_gated_desc& d, bool bwd, int col0, Plan* out) {
    constexpr int SPL = Form<T>::SPL, KC = Form<T>::KC;
    Plan p{};
    p.C = d.channels;
    p.H = d.hidden;
    p.O = d.out_channels;
    p.Kx = up16(p.C);
    p.Ky = bwd ? up16(p.O) : 0;
    p.col0 = col0;
    p.cols = imin((bwd ? p.C : p.O) - col0, SPL == 3 ? 128 : 256);
    p.N2 = up16(p.cols);
    const int most = bwd && p.N2 * (SPL == 3 ? 2 : 1) > 128 ? 32 : 64;
    p.nJ = (p.H + most - 1) / most;
    p.NH = up16((p.H + p.nJ - 1) / p.nJ);
    p.per = SPL == 3 ? imin(p.nJ, std::max(1, kRunSteps / (p.NH / 16 * (bwd ? 2 : 1)))) : p.nJ;
    p.runs = (p.nJ + p.per - 1) / p.per;
    const int w1 = (bwd ? 3 : 2) * p.NH, w2 = p.N2 * (SPL == 3 ? 2 : 1);
    p.n_d1 = 3 * w1 + w2 <= 512 ? 3 : 2;
    p.n_d2 = p.n_d1 * w1 + 2 * w2 <= 512 ? 2 : 1;
    p.nKx = (p.Kx + KC - 1) / KC;
    p.nKy = (p.Ky + KC - 1) / KC;
    p.nH = (p.NH + KC - 1) / KC;
    const int kx = imin(KC, std::max(p.Kx, p.Ky)), kh = imin(KC, p.NH);
    p.a_slot = (kx / 16) * 16 * kAGroup * SPL;
    p.b_slot = std::max(2 * p.NH * imin(KC, p.Kx), std::max(p.NH * imin(KC, p.Ky), p.N2 * kh)) * 2 * SPL;
    p.job_bytes = (p.NH * (2 * p.Kx + p.Ky) + (bwd ? 2 : 1) * p.N2 * p.NH) * 2 * SPL;
    const int vec = (2 * p.NH * p.nJ + p.N2) * 4;
    p.vec_smem = vec <= 8192;  // hidden widths up to about 1000; wider ones read them from L1 or L2
    const int64_t room = kSmem - 1024 - (int64_t)sizeof(Bars) - (p.vec_smem ? vec : 0);
    const int64_t all = (int64_t)p.nJ * p.job_bytes;
    const int nA = p.nKx + p.nKy;
    int64_t bytes;
    if (all + 2 * p.a_slot <= room) {
        p.resident = 1;
        p.nb = 1;
        p.na = (int)std::min<int64_t>(kMaxA, (room - all) / p.a_slot);
        bytes = all;
    } else {
        p.nb = 2;
        if (2 * p.a_slot + 2 * (int64_t)p.b_slot > room) return false;
        // spare room: first for as many A pieces as a tile has, then for weights
        p.na = 2;
        while (p.na < kMaxA && p.na < nA && (p.na + 1) * p.a_slot + 2 * (int64_t)p.b_slot <= room) ++p.na;
        while (p.nb < 6 && p.na * p.a_slot + (p.nb + 1) * (int64_t)p.b_slot <= room) ++p.nb;
        while (p.na < kMaxA && (p.na + 1) * p.a_slot + p.nb * (int64_t)p.b_slot <= room) ++p.na;
        bytes = (int64_t)p.nb * p.b_slot;
    }
    p.reuse = p.nJ > 1 && p.na >= nA;
    p.o_a = 0;
    p.o_b = p.na * p.a_slot;
    p.o_b = (p.o_b + 127) & ~127;
    p.o_vec = (int)((p.o_b + bytes + 127) & ~127);
    p.o_bar = (p.o_vec + (p.vec_smem ? vec : 0) + 127) & ~127;
    p.smem = std::max(p.o_bar + (int)sizeof(Bars), 120 * 1024);  // one CTA an SM: it holds the whole tensor memory
    *out = p;
    return p.smem <= kSmem;
}

constexpr const char* kTooLarge = "these channel counts do not fit a CTA's shared memory";

struct Sizes {
    size_t packed, vec, z, partial, sums, bytes;
    int64_t slab_tiles, tiles;
    int splits, wtiles;
};

// weights: the backward leaves gradients of the weights or the biases, beside or without dL/dx
template <class T>
Sizes sizes_of(const nop_gated_desc& d, const Plan& p, bool bwd, bool weights) {
    auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
    Sizes s{};
    s.tiles = ceil_div(d.batch * d.points, TP);
    size_t at = 0, images = 0, vectors = 0;
    for (Plan q = p;;) {  // the launches of a call use the same places in turn
        images = std::max(images, (size_t)q.nJ * q.job_bytes);
        vectors = std::max(vectors, (size_t)(2 * q.NH * q.nJ + q.N2) * 4);
        if (q.col0 + q.cols >= (bwd ? q.C : q.O) || !make_plan<T>(d, bwd, q.col0 + q.cols, &q)) break;
    }
    s.packed = at;
    at += up(images);
    s.vec = at;
    at += up(vectors);
    if (weights) {
        // The scratch of a slab: up to 512 MB, in whole waves of 148 tiles, and at least one wave (512 MB at a hidden width of
        // some 2300, 3.8 GB at 16384 with 256 channels).  Slabs that stay in L2 save the scratch's
        // trip through HBM but lose more to their launches' beginnings and ends: 64 MB slabs took 2207 us where
        // 512 MB take 1646 (fp32, 64 channels, hidden 128, 2^20 points), and larger ones 1626.
        using Z = typename Scratch<T>::type;
        const int64_t tile_bytes = (int64_t)(3 * Scratch<T>::PARTS * p.H + p.C + p.O) * TP * sizeof(Z);
        const int64_t waves = std::max<int64_t>(1, (int64_t)(512 << 20) / (148 * tile_bytes));
        s.slab_tiles = std::min<int64_t>(s.tiles, 148 * waves);
        s.wtiles = (int)(ceil_div(2 * p.H, 128) * ceil_div(p.C, 128) + ceil_div(p.H, 128) * ceil_div(p.O, 128));
        const int64_t pieces = s.slab_tiles * (TP / WForm<Z>::KC);
        s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(148 / s.wtiles, pieces));
        s.z = at;
        at += up((size_t)s.slab_tiles * tile_bytes);
        s.partial = at;
        at += up((size_t)s.splits * s.wtiles * 128 * 128 * 4);
        s.sums = at;
        at += up((size_t)s.splits * (2 * p.H + p.O) * 8);
    }
    s.bytes = at;
    return s;
}

int32_t check(const nop_gated_desc* d) {
    if (!d) return fail(NOP_E_INVALID, "descriptor is NULL");
    if (d->abi_version != NOP_ABI_VERSION) return fail(NOP_E_INVALID, "ABI version mismatch");
    if (d->dtype < NOP_DTYPE_FP32 || d->dtype > NOP_DTYPE_FP16) return fail(NOP_E_INVALID, "unknown dtype");
    if (d->x_dtype != d->dtype && d->x_dtype != NOP_DTYPE_E4M3)
        return fail(NOP_E_INVALID, "x has the weights' type, or e4m3");
    if (d->x_dtype == NOP_DTYPE_E4M3 && d->dtype == NOP_DTYPE_FP32)
        return fail(NOP_E_UNSUPPORTED, "an e4m3 field needs bf16 or fp16 weights");
    if (d->activation != NOP_ACT_SILU && d->activation != NOP_ACT_GELU) return fail(NOP_E_INVALID, "unknown activation");
    if (d->batch < 0 || d->points < 0) return fail(NOP_E_INVALID, "batch and points must be >= 0");
    if (d->channels < 1 || d->hidden < 1 || d->out_channels < 1)
        return fail(NOP_E_INVALID, "channels, hidden and out_channels must be positive");
    if (d->channels > 256 || d->out_channels > 256)
        return fail(NOP_E_UNSUPPORTED, "more than 256 channels are not supported");
    if (d->hidden > 16384) return fail(NOP_E_UNSUPPORTED, "a hidden width above 16384 is not supported");
    if (d->points && d->batch > (int64_t)0x7fffff00LL / d->points)
        return fail(NOP_E_UNSUPPORTED, "more than 2^31 points");
    return NOP_OK;
}

template <class F>
int32_t by_type(int dtype, F&& f) {
    if (dtype == NOP_DTYPE_FP32) return f(float{});
    if (dtype == NOP_DTYPE_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}

struct Device {
    int dev = 0, sms = 148;
    int* status = nullptr;
};
int32_t device(Device* d) {
    const int32_t rc = current_device(&d->dev, &d->sms);
    if (rc != NOP_OK) return rc;
    d->status = status_word(d->dev);
    if (!d->status) return fail(NOP_E_CUDA, "status word of the tensor-core kernels is not available");
    return NOP_OK;
}

template <auto KERNEL, class... A>
int32_t launch(const Device& d, unsigned grid, int threads, int smem, cudaStream_t s, A... args) {
    const int32_t rc = allow_smem<KERNEL>(d.dev, kSmem);
    if (rc != NOP_OK) return rc;
    KERNEL<<<grid, threads, smem, s>>>(args...);
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// `rows` rows of `points` points, boxes of 128 bytes x `box` rows
template <class T>
bool row_map(CUtensorMap* m, void* base, int64_t points, int64_t rows, int box) {
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encoder());
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)points, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)points * sizeof(T)};
    const cuuint32_t sizes[2] = {(cuuint32_t)(128 / sizeof(T)), (cuuint32_t)box};
    const cuuint32_t ones[2] = {1, 1};
    const CUtensorMapDataType type = std::is_same<T, float>::value    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return enc(m, type, 2, base, dims, strides, sizes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool aligned(std::initializer_list<const void*> ps, uintptr_t to) {
    uintptr_t all = 0;
    for (const void* p : ps) all |= (uintptr_t)p;
    return all % to == 0;
}

template <class T, bool BWD>
int32_t pack(const Plan& p, const nop_gated_operands& o, const Sizes& z, char* ws, cudaStream_t s) {
    const int items = (int)(((int64_t)p.nJ * p.job_bytes) / (16 * Form<T>::SPL));
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(items, 256), 592);
    k_pack<T, BWD><<<grid, 256, 0, s>>>(p, static_cast<const T*>(o.w_gate), static_cast<const T*>(o.w_up),
                                        static_cast<const T*>(o.w_down), static_cast<const T*>(o.b_gate),
                                        static_cast<const T*>(o.b_up), static_cast<const T*>(o.b_down),
                                        ws + z.packed, reinterpret_cast<float*>(ws + z.vec));
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

template <class T>
Params params_of(const nop_gated_desc& d, const Plan& p, const nop_gated_operands& o, const Sizes& z, char* ws) {
    Params q{};
    q.x = o.x;
    q.scale = o.x_scale;
    q.packed = ws + z.packed;
    q.bias = reinterpret_cast<const float*>(ws + z.vec);
    q.P = (uint32_t)d.points;
    q.points = (uint32_t)(d.batch * d.points);
    uint32_t s = 0;
    while ((1ull << s) < d.points) ++s;
    q.p_shift = 31 + s;
    q.p_mul = (uint32_t)(((1ull << q.p_shift) + d.points - 1) / d.points);
    q.tiles = (int)z.tiles;
    q.pl = p;
    return q;
}

template <class T, class IN>
int32_t forward(const nop_gated_desc& d, Plan p, const nop_gated_operands& o, const Sizes& z, char* ws, cudaStream_t s) {
    Device dev;
    int32_t rc = device(&dev);
    if (rc != NOP_OK) return rc;
    const unsigned grid = (unsigned)std::min<int64_t>(z.tiles, dev.sms);
    while (true) {
        if ((rc = pack<T, false>(p, o, z, ws, s)) != NOP_OK) return rc;
        Params q = params_of<T>(d, p, o, z, ws);
        q.out = o.y;
        q.vec = d.points % 4 == 0 && aligned({o.x}, 4 * sizeof(IN));
        rc = d.activation == NOP_ACT_GELU
                 ? launch<k_block<T, IN, false, true>>(dev, grid, kThreads, p.smem, s, q, dev.status)
                 : launch<k_block<T, IN, false, false>>(dev, grid, kThreads, p.smem, s, q, dev.status);
        if (rc != NOP_OK || p.col0 + p.cols >= p.O) return rc;
        if (!make_plan<T>(d, false, p.col0 + p.cols, &p)) return fail(NOP_E_UNSUPPORTED, kTooLarge);
    }
}

bool of_weights(const nop_gated_grads& g) {
    return g.gw_gate || g.gw_up || g.gw_down || g.gb_gate || g.gb_up || g.gb_down;
}

template <class T>
int32_t backward(const nop_gated_desc& d, Plan p, const nop_gated_operands& o, const nop_gated_grads& g,
                 const Sizes& z, char* ws, cudaStream_t s) {
    Device dev;
    int32_t rc = device(&dev);
    if (rc != NOP_OK) return rc;
    if ((rc = pack<T, true>(p, o, z, ws, s)) != NOP_OK) return rc;
    const bool weights = of_weights(g);
    Params q = params_of<T>(d, p, o, z, ws);
    q.gy = g.gy;
    q.out = g.gx;
    q.z = weights ? ws + z.z : nullptr;
    q.vec = d.points % 4 == 0 && aligned({o.x, g.gy}, 4 * sizeof(T));
    WParams w{};
    w.partial = reinterpret_cast<float*>(ws + z.partial);
    w.sums = g.gb_gate || g.gb_up || g.gb_down ? reinterpret_cast<double*>(ws + z.sums) : nullptr;
    w.C = p.C;
    w.H = p.H;
    w.O = p.O;
    using Z = typename Scratch<T>::type;
    // x and e in place: of the scratch's type, whole tiles a sample, on 16-byte boundaries
    const bool in_place = std::is_same<Z, T>::value && d.points % TP == 0 && aligned({o.x, g.gy}, 16);
    w.rows = 3 * Scratch<T>::PARTS * p.H + (in_place ? 0 : p.C + p.O);
    w.per_sample = in_place ? (int)(d.points / TP) : 0;
    q.z_rows = w.rows;
    w.nC = (int)ceil_div(p.C, 128);
    w.nO = (int)ceil_div(p.O, 128);
    w.mX = (int)ceil_div(2 * p.H, 128);
    w.mH = (int)ceil_div(p.H, 128);
    w.splits = z.splits;
    CUtensorMap mg{}, mh{}, mx{}, me{};
    if (weights) {
        const int64_t rows = z.slab_tiles * w.rows;
        void *xs = ws + z.z, *es = ws + z.z;
        if (in_place) {
            xs = const_cast<void*>(o.x);
            es = const_cast<void*>(g.gy);
        }
        if (!(row_map<Z>(&mg, ws + z.z, TP, rows, imin(128, 2 * p.H)) &&
              row_map<Z>(&mh, ws + z.z, TP, rows, imin(128, p.H)) &&
              row_map<Z>(&mx, xs, in_place ? d.points : TP, in_place ? d.batch * p.C : rows, imin(128, p.C)) &&
              row_map<Z>(&me, es, in_place ? d.points : TP, in_place ? d.batch * p.O : rows, imin(128, p.O))))
            return fail(NOP_E_CUDA, "cuTensorMapEncodeTiled failed");
    }
    const int64_t slab = weights ? z.slab_tiles : z.tiles;
    for (int64_t t = 0; t < z.tiles; t += slab) {
        q.tile0 = (int)t;
        q.tiles = (int)std::min<int64_t>(slab, z.tiles - t);
        const unsigned grid = (unsigned)std::min<int64_t>(q.tiles, dev.sms);
        rc = d.activation == NOP_ACT_GELU ? launch<k_block<T, T, true, true>>(dev, grid, kThreads, p.smem, s, q, dev.status)
                                          : launch<k_block<T, T, true, false>>(dev, grid, kThreads, p.smem, s, q, dev.status);
        if (rc != NOP_OK) return rc;
        if (!weights) continue;
        w.tile0 = (int)t;
        w.accumulate = t > 0;
        using F = WForm<Z>;
        w.pieces = q.tiles * (TP / F::KC);
        rc = launch<k_wgrad<Z>>(dev, (unsigned)(z.splits * z.wtiles), F::THREADS, F::BODY + (int)sizeof(WBars), s, mg, mh, mx,
                                me, w, dev.status);
        if (rc != NOP_OK) return rc;
    }
    // dL/dx of the channels past the first launch's: the products again, without the scratch
    while (g.gx && p.col0 + p.cols < p.C) {
        if (!make_plan<T>(d, true, p.col0 + p.cols, &p)) return fail(NOP_E_UNSUPPORTED, kTooLarge);
        if ((rc = pack<T, true>(p, o, z, ws, s)) != NOP_OK) return rc;
        Params r = params_of<T>(d, p, o, z, ws);
        r.gy = q.gy;
        r.out = q.out;
        r.vec = q.vec;
        const unsigned grid = (unsigned)std::min<int64_t>(z.tiles, dev.sms);
        rc = d.activation == NOP_ACT_GELU ? launch<k_block<T, T, true, true>>(dev, grid, kThreads, p.smem, s, r, dev.status)
                                          : launch<k_block<T, T, true, false>>(dev, grid, kThreads, p.smem, s, r, dev.status);
        if (rc != NOP_OK) return rc;
    }
    if (!weights) return NOP_OK;
    const unsigned vecs = w.sums ? (unsigned)ceil_div(2 * p.H + p.O, 128) : 0;
    k_finish<T><<<3 * p.H + vecs, 128, 0, s>>>(w, static_cast<T*>(g.gw_gate), static_cast<T*>(g.gw_up),
                                               static_cast<T*>(g.gw_down), static_cast<T*>(g.gb_gate),
                                               static_cast<T*>(g.gb_up), static_cast<T*>(g.gb_down));
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

int32_t check_operands(const nop_gated_desc& d, const nop_gated_operands* o) {
    if (!o) return fail(NOP_E_INVALID, "operands are NULL");
    if (!o->x || !o->w_gate || !o->w_up || !o->w_down)
        return fail(NOP_E_INVALID, "x, w_gate, w_up and w_down must be non-NULL");
    if (d.x_dtype == NOP_DTYPE_E4M3 && !o->x_scale) return fail(NOP_E_INVALID, "an e4m3 field needs x_scale");
    const uintptr_t size = d.dtype == NOP_DTYPE_FP32 ? 4 : 2;
    if ((d.x_dtype != NOP_DTYPE_E4M3 && (uintptr_t)o->x % size) || (uintptr_t)o->x_scale % 4 ||
        !aligned({o->w_gate, o->w_up, o->w_down, o->b_gate, o->b_up, o->b_down, o->y}, size))
        return fail(NOP_E_ALIGNMENT, "a pointer is not aligned to its type");
    return NOP_OK;
}

}  // namespace gated
}  // namespace nop

using namespace nop;

extern "C" {

int32_t nop_gated_workspace_size(const nop_gated_desc* d, int32_t backward, size_t* bytes) {
    const int32_t rc = gated::check(d);
    if (rc != NOP_OK) return rc;
    if (!bytes) return fail(NOP_E_INVALID, "bytes is NULL");
    if (backward < 0 || backward > 2) return fail(NOP_E_INVALID, "the pass must be 0, 1 or 2");
    return gated::by_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        gated::Plan p;
        if (!gated::make_plan<T>(*d, backward != 0, 0, &p))
            return fail(NOP_E_UNSUPPORTED, gated::kTooLarge);
        *bytes = gated::sizes_of<T>(*d, p, backward != 0, backward == 1).bytes;
        return (int32_t)NOP_OK;
    });
}

int32_t nop_gated_forward(const nop_gated_desc* d, const nop_gated_operands* o, void* workspace, size_t workspace_bytes,
                          void* stream) {
    int32_t rc = gated::check(d);
    if (rc != NOP_OK) return rc;
    if (d->batch == 0 || d->points == 0) return NOP_OK;
    if ((rc = gated::check_operands(*d, o)) != NOP_OK) return rc;
    if (!o->y) return fail(NOP_E_INVALID, "y must be non-NULL");
    return gated::by_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        gated::Plan p;
        if (!gated::make_plan<T>(*d, false, 0, &p))
            return fail(NOP_E_UNSUPPORTED, gated::kTooLarge);
        const gated::Sizes z = gated::sizes_of<T>(*d, p, false, false);
        if (!workspace || workspace_bytes < z.bytes) return fail(NOP_E_WORKSPACE, "workspace missing or too small");
        if ((uintptr_t)workspace % 256) return fail(NOP_E_ALIGNMENT, "the workspace must be 256-byte aligned");
        char* ws = static_cast<char*>(workspace);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if constexpr (sizeof(T) == 2) {
            if (d->x_dtype == NOP_DTYPE_E4M3) return gated::forward<T, uint8_t>(*d, p, *o, z, ws, s);
        }
        return gated::forward<T, T>(*d, p, *o, z, ws, s);
    });
}

int32_t nop_gated_backward(const nop_gated_desc* d, const nop_gated_operands* o, const nop_gated_grads* g,
                           void* workspace, size_t workspace_bytes, void* stream) {
    int32_t rc = gated::check(d);
    if (rc != NOP_OK) return rc;
    if (d->x_dtype != d->dtype) return fail(NOP_E_UNSUPPORTED, "the backward takes no e4m3 field");
    if (!g) return fail(NOP_E_INVALID, "grads are NULL");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->batch == 0 || d->points == 0) {  // no points: the weights' gradients are zero
        const size_t size = d->dtype == NOP_DTYPE_FP32 ? 4 : 2;
        const size_t h = d->hidden, c = d->channels, n = d->out_channels;
        for (auto [ptr, count] : {std::pair<void*, size_t>{g->gw_gate, h * c}, {g->gw_up, h * c}, {g->gw_down, n * h},
                                  {g->gb_gate, h}, {g->gb_up, h}, {g->gb_down, n}})
            if (ptr) NOP_CUDA_TRY(cudaMemsetAsync(ptr, 0, count * size, s));
        return NOP_OK;
    }
    if ((rc = gated::check_operands(*d, o)) != NOP_OK) return rc;
    if (!g->gy) return fail(NOP_E_INVALID, "gy must be non-NULL");
    if (!gated::aligned({g->gy, g->gx, g->gw_gate, g->gw_up, g->gw_down, g->gb_gate, g->gb_up, g->gb_down},
                        d->dtype == NOP_DTYPE_FP32 ? 4 : 2))
        return fail(NOP_E_ALIGNMENT, "a pointer is not aligned to its type");
    return gated::by_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        gated::Plan p;
        if (!gated::make_plan<T>(*d, true, 0, &p))
            return fail(NOP_E_UNSUPPORTED, gated::kTooLarge);
        const gated::Sizes z = gated::sizes_of<T>(*d, p, true, gated::of_weights(*g));
        if (!workspace || workspace_bytes < z.bytes) return fail(NOP_E_WORKSPACE, "workspace missing or too small");
        if ((uintptr_t)workspace % 256) return fail(NOP_E_ALIGNMENT, "the workspace must be 256-byte aligned");
        return gated::backward<T>(*d, p, *o, *g, z, static_cast<char*>(workspace), s);
    });
}

}  // extern "C"
