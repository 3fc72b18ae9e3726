// Root-mean-square norm over the channels of every point, with the residual's addition.
//
//   r = x + res (rounded to the field's type),  inv = 1 / sqrt(mean_c r^2 + eps),  y_c = r_c inv w_c
//
// on fields [B, C, P] (P points per sample).  Backward, with g = dL/dy and gr = dL/dr from the residual's path:
//
//   dL/dr_c = inv (g_c w_c - r_c inv m) + gr_c,  m = mean_c(g_c w_c r_c inv),   dL/dw_c = sum_points g_c r_c inv
//
// and x and res share dL/dr.  The statistics are fp32 sums over the channels of a point.
//
// 8-bit output: q_c = e4m3(y_c / s) with one scale a point, the least power of two with max_c |y_c| <= 448 s
// (448 is e4m3's largest value).  A power of two costs e4m3 nothing, its steps being relative, and q s has four
// significant bits, so it is exact in bf16 and fp32.
//
// Bound: HBM, one pass over every field.  The channels of a point lie P values apart, so a warp takes 32 V
// neighbouring points (V values a thread in one load of up to 16 bytes) of some channels, and W warps share the
// channels of the same points: warp k holds channels k, k + W, ... (at most NC) in registers between the sums
// and the scaling, and the W partial sums meet in shared memory.  More than 256 channels do not fit the
// registers of a CTA: the second pass then reads the tile again, out of L2.
//
// Measured on B200, 64 channels x 2^21 points fp32, of the measured copy bandwidth: forward 193 us (86%), with the
// residual 342 us (97%), backward 406 us (61%) and 442 us with the residual's gradient (75%; two fields in registers and
// a meeting of the warps between them and the output).  Rows that are not aligned load one value a thread: 55 to 80% in
// fp32, 25 to 40% in bf16, whose two-byte loads keep too few bytes in flight.
#include "nop_internal.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

namespace nop {
namespace rms {

constexpr int kMaxWarps = 16;

// V values of type T as they move between memory and registers, in 32-bit words: 16-bit values are cut out of them by
// shifts (through a union with an array they went to local memory, and a bf16 call took as long as an fp32 one)
template <class T, int V>
struct Vec {
    static constexpr int BYTES = V * (int)sizeof(T), WORDS = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (BYTES == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (BYTES == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (BYTES == 8) {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            w[0] = q.x;
            w[1] = q.y;
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            w[0] = q.x;
            w[1] = q.y;
            w[2] = q.z;
            w[3] = q.w;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYTES == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
        else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
    }
    __device__ __forceinline__ void put(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const float hi = 2 * i + 1 < V ? v[(2 * i + 1) % V] : 0.f;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(v[2 * i], hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        }
    }
};

// the least power of two s with most <= 448 s, 448 = 0.875 2^9 (1 for a point of zeros, and for one whose
// values are not finite; not below the smallest normal number)
__device__ __forceinline__ float e4m3_scale(float most) {
    if (!(most > 0.f) || !(most < INFINITY)) return 1.f;
    int e;
    const float m = frexpf(most, &e);
    e -= m <= 0.875f ? 9 : 8;
    return ldexpf(1.f, e < -126 ? -126 : e);
}

__device__ __forceinline__ uint8_t to_e4m3(float v) {
    // NaN and infinity become NaN; a value that rounds past 448 by the last bit of the scaling saturates
    return fabsf(v) < INFINITY ? __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3) : (uint8_t)0x7f;
}

// Threads a CTA has at most, and the CTAs an SM is to hold at least: registers for the NC (with the residual twice as
// many) loads of up to four words that a thread has in flight, and as many warps as that leaves.
constexpr int threads_of(int nc) { return nc == 8 ? 256 : 512; }
constexpr int fwd_ctas(int nc, int words, bool res) {
    return nc == 8 ? (words == 4 ? (res ? 3 : 4) : words == 2 ? 4 : 6) : nc == 16 ? (words == 1 ? 2 : 1) : 2;
}
constexpr int bwd_ctas(int nc, int words) { return nc == 8 ? (words == 1 ? 4 : 3) : nc == 16 ? 1 : 2; }

struct Args {
    const void *x, *res, *gy, *gr;
    const float* w;
    void *y, *r, *gx;
    uint8_t* q;
    float *scale, *partial;
    int C, W;          // channels, warps that share a tile's channels
    int64_t P, groups; // points per sample, vectors of V points
    float eps;
    int64_t tiles;     // 32 vectors each
};

// position of vector g: offset of its first point's first channel
template <int V>
__device__ __forceinline__ int64_t base_of(const Args& a, int64_t g) {
    const int64_t n = g * V, b = n / a.P;
    return b * a.C * a.P + (n - b * a.P);
}

// every warp's V sums of its slot's tile added up (the slot's W warps in order)
template <int V>
__device__ __forceinline__ void meet(float (&s)[V], float* red, int warp, int lane, int W, bool maximum) {
#pragma unroll
    for (int j = 0; j < V; ++j) red[(warp * V + j) * 32 + lane] = s[j];
    __syncthreads();
    const int w0 = warp / W * W;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float t = red[(w0 * V + j) * 32 + lane];
        for (int k = 1; k < W; ++k) {
            const float u = red[((w0 + k) * V + j) * 32 + lane];
            t = maximum ? ((u > t || u != u) ? u : t) : t + u;
        }
        s[j] = t;
    }
}

// RES: 0 no residual, 1 with it.  Q8: the output in 8 bits.  NC: channels a warp holds in registers, 0: none are
// held and the second pass reads the tile again.
template <class T, int V, int NC, bool RES, bool Q8>
__global__ void __launch_bounds__(threads_of(NC), fwd_ctas(NC, Vec<T, V>::WORDS, RES)) k_fwd(const Args a) {
    extern __shared__ float red[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W;
    const int slots = (int)(blockDim.x >> 5) / W;
    const int cw = warp % W;
    const int64_t g = ((int64_t)blockIdx.x * slots + warp / W) * 32 + lane;
    const bool valid = g < a.groups;
    const int64_t base = valid ? base_of<V>(a, g) : 0;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* res = static_cast<const T*>(a.res) + base;
    T* r = static_cast<T*>(a.r) + base;
    constexpr int N = NC ? NC : 1;
    Vec<T, V> f[N];
    float s[V], m[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = m[j] = 0.f;

    auto sum_up = [&](Vec<T, V>& v, const Vec<T, V>& u, int c) {
        if (RES) {
            float t[V];
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = v.get(j) + u.get(j);
            v.put(t);
            v.store(r + c * a.P);
        }
        const float w = Q8 && a.w ? __ldg(a.w + c) : 1.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float t = v.get(j);
            s[j] = fmaf(t, t, s[j]);
            if (Q8) {
                const float p = fabsf(t * w);
                m[j] = (p > m[j] || p != p) ? p : m[j];
            }
        }
    };
    if constexpr (NC > 0) {
        // eight channels at a time: the residual's registers are free again for the next eight
#pragma unroll
        for (int i0 = 0; i0 < N; i0 += 8) {
            Vec<T, V> u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = cw + (i0 + i) * W;
                if (valid && c < a.C) {
                    f[i0 + i].load(x + c * a.P);
                    if (RES) u[i].load(res + c * a.P);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = cw + (i0 + i) * W;
                if (valid && c < a.C) sum_up(f[i0 + i], u[i], c);
            }
        }
    } else if (valid) {
#pragma unroll 4
        for (int c = cw; c < a.C; c += W) {
            Vec<T, V> v, u;
            v.load(x + c * a.P);
            if (RES) u.load(res + c * a.P);
            sum_up(v, u, c);
        }
    }
    meet<V>(s, red, warp, lane, W, false);
    float inv[V], qs[V];
#pragma unroll
    for (int j = 0; j < V; ++j) inv[j] = 1.f / sqrtf(s[j] / (float)a.C + a.eps);
    if constexpr (Q8) {
        meet<V>(m, red + (blockDim.x >> 5) * 32 * V, warp, lane, W, true);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float sc = e4m3_scale(m[j] * inv[j]);
            qs[j] = 1.f / sc;  // exact: a power of two
            if (valid && cw == 0) {
                const int64_t n = g * V + j;  // scale is [B, 1, P]
                a.scale[n] = sc;
            }
        }
    }
    if (!valid) return;
    auto finish = [&](const Vec<T, V>& v, int c) {
        const float w = a.w ? __ldg(a.w + c) : 1.f;
        if constexpr (Q8) {
            uint32_t o[(V + 3) / 4] = {};
#pragma unroll
            for (int j = 0; j < V; ++j) o[j / 4] |= (uint32_t)to_e4m3(v.get(j) * inv[j] * w * qs[j]) << (8 * (j % 4));
            uint8_t* to = a.q + base + c * a.P;
            if constexpr (V == 1) *to = (uint8_t)o[0];
            else if constexpr (V == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)o[0];
            else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(to) = o[0];
            else *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
        } else {
            float t[V];
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = v.get(j) * inv[j] * w;
            Vec<T, V> o;
            o.put(t);
            o.store(static_cast<T*>(a.y) + base + c * a.P);
        }
    };
    if constexpr (NC > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = cw + i * W;
            if (c < a.C) finish(f[i], c);
        }
    } else {
#pragma unroll 4
        for (int c = cw; c < a.C; c += W) {
            Vec<T, V> v;
            v.load((RES ? r : x) + c * a.P);
            finish(v, c);
        }
    }
}

// Backward.  A CTA walks the tiles blockIdx.x * slots + slot, + gridDim.x * slots, ...; each thread keeps the
// sums of dL/dw of its channels over all its points and the warp's lanes meet once at the end, so that the
// partial sums [slot of the grid][C] are few and are added in a fixed order (k_reduce).  NC = 0: the channels'
// sums are kept in shared memory (one warp owns a channel) and the lanes meet in every tile.
template <class T, int V, int NC, bool GR>
__global__ void __launch_bounds__(threads_of(NC), bwd_ctas(NC, Vec<T, V>::WORDS)) k_bwd(const Args a) {
    extern __shared__ float red[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W, warps = blockDim.x >> 5;
    const int slots = warps / W, slot = warp / W, cw = warp % W;
    float* gw_sum = red + 4 * warps * 32 * V;  // NC = 0: [C]
    if (NC == 0) {
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) gw_sum[c] = 0.f;
        __syncthreads();
    }
    constexpr int N = NC ? NC : 1;
    constexpr bool kHoldR = NC == 8;  // dL/dr of the residual's path comes with the first loads (registers for 8 channels)
    float gw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) gw[i] = 0.f;
    const T* px = static_cast<const T*>(a.x);
    const T* pg = static_cast<const T*>(a.gy);
    const T* pr = static_cast<const T*>(a.gr);
    T* po = static_cast<T*>(a.gx);
    int turn = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * slots; t0 < a.tiles; t0 += (int64_t)gridDim.x * slots, turn ^= 1) {
        const int64_t g = (t0 + slot) * 32 + lane;
        const bool valid = g < a.groups;
        const int64_t base = valid ? base_of<V>(a, g) : 0;
        Vec<T, V> f[N], d[N], r[N];
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
        auto sum_up = [&](const Vec<T, V>& v, const Vec<T, V>& e, int c) {
            const float w = a.w ? __ldg(a.w + c) : 1.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1[j] = fmaf(v.get(j), v.get(j), s1[j]);
                s2[j] = fmaf(e.get(j) * w, v.get(j), s2[j]);
            }
        };
        if constexpr (NC > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = cw + i * W;
                if (valid && c < a.C) {
                    f[i].load(px + base + c * a.P);
                    d[i].load(pg + base + c * a.P);
                    if (GR && kHoldR) r[i].load(pr + base + c * a.P);
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = cw + i * W;
                if (valid && c < a.C) sum_up(f[i], d[i], c);
            }
        } else if (valid) {
#pragma unroll 4
            for (int c = cw; c < a.C; c += W) {
                Vec<T, V> v, e;
                v.load(px + base + c * a.P);
                e.load(pg + base + c * a.P);
                sum_up(v, e, c);
            }
        }
        // two buffers in turn: the next tile's sums are written while slower warps still read these
        float* red1 = red + turn * 2 * warps * 32 * V;
        float* red2 = red1 + warps * 32 * V;
#pragma unroll
        for (int j = 0; j < V; ++j) red2[(warp * V + j) * 32 + lane] = s2[j];
        meet<V>(s1, red1, warp, lane, W, false);
        const int w0 = slot * W;
        float inv[V], back[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float t = red2[(w0 * V + j) * 32 + lane];
            for (int k = 1; k < W; ++k) t += red2[((w0 + k) * V + j) * 32 + lane];
            inv[j] = 1.f / sqrtf(s1[j] / (float)a.C + a.eps);
            back[j] = inv[j] * inv[j] * (t / (float)a.C);  // inv m
        }
        auto finish = [&](const Vec<T, V>& v, const Vec<T, V>& e, Vec<T, V> u, int c) -> float {
            const float w = a.w ? __ldg(a.w + c) : 1.f;
            float q[V];
            if (GR && !kHoldR) u.load(pr + base + c * a.P);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sum = fmaf(e.get(j), v.get(j) * inv[j], sum);
                const float t = inv[j] * (e.get(j) * w - v.get(j) * back[j]);
                q[j] = GR ? t + u.get(j) : t;
            }
            Vec<T, V> o;
            o.put(q);
            if (po) o.store(po + base + c * a.P);
            return sum;
        };
        if constexpr (NC > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = cw + i * W;
                if (valid && c < a.C) gw[i] += finish(f[i], d[i], r[i], c);
            }
        } else {
            for (int c = cw; c < a.C; c += W) {
                float sum = 0.f;
                if (valid) {
                    Vec<T, V> v, e;
                    v.load(px + base + c * a.P);
                    e.load(pg + base + c * a.P);
                    sum = finish(v, e, Vec<T, V>(), c);
                }
                if (a.partial) {
#pragma unroll
                    for (int o = 16; o; o >>= 1) sum += __shfl_down_sync(0xffffffffu, sum, o);
                    if (lane == 0) gw_sum[c] += sum;
                }
            }
        }
    }
    if (!a.partial) return;
    const int64_t row = (int64_t)blockIdx.x * slots + slot, rows = (int64_t)gridDim.x * slots;
    if constexpr (NC > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = cw + i * W;
            float v = gw[i];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
            if (lane == 0 && c < a.C) a.partial[c * rows + row] = v;
        }
    } else {
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) a.partial[c * rows + row] = gw_sum[c];
    }
}

// dL/dw_c = the grid's partial sums of channel c, added in 64 bits in a fixed order
__global__ void __launch_bounds__(128) k_reduce(const float* __restrict__ partial, int rows, float* __restrict__ gw) {
    __shared__ double part[4];
    const float* p = partial + (int64_t)blockIdx.x * rows;
    double s = 0.0;
    for (int i = threadIdx.x; i < rows; i += 128) s += (double)p[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_down_sync(0xffffffffu, s, o);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) gw[blockIdx.x] = (float)(part[0] + part[1] + part[2] + part[3]);
}

constexpr int kMaxChannels = 8192;   // the backward's shared-memory sums
constexpr int kMaxSms = 160;         // CTAs are planned for at most so many multiprocessors

// How a call is cut: V points a thread, W warps a tile, NC channels a warp.
struct Cut {
    int V, W, NC, warps;
    int64_t groups, tiles;
    // the backward's CTAs: with 8 channels a warp a few times what an SM holds, so that the last ones to end are a small
    // part (12 an SM against 4: 557 -> 444 us at 64 channels, 2^21 points); with 16 the sums at a CTA's end cost more
    int max_grid(int sms) const { return (sms < kMaxSms ? sms : kMaxSms) * (NC == 8 ? 12 : warps > 8 ? 2 : 4); }
};

// V: the widest load of up to 16 bytes that the points per sample and every pointer allow; one point a thread
// when that would leave most SMs without a tile.  W x NC covers the channels.
Cut cut_of(const nop_norm_desc& d, int size, bool aligned, int sms, bool backward) {
    Cut c{};
    const int64_t points = d.batch * d.points;
    int v = 1;
    // the backward holds two fields: half as many values a thread
    const int most = size == 4 ? (backward ? 2 : 4) : (backward ? 4 : 8);
    if (aligned)
        for (int k = most; k > 1; k /= 2)
            if (d.points % k == 0) {
                v = k;
                break;
            }
    if (ceil_div(points, 32 * v) < 2 * sms) v = 1;
    c.V = v;
    if (d.channels <= 64) {
        c.NC = 8;
        for (c.W = 1; c.W * c.NC < d.channels; c.W *= 2) {}
    } else {
        c.NC = 16;
        c.W = d.channels <= 128 ? 8 : 16;
        if (d.channels > 256) c.NC = 0;
    }
    c.warps = c.W > 8 ? c.W : 8;
    c.groups = points / v;
    c.tiles = ceil_div(c.groups, 32);
    return c;
}

int32_t check(const nop_norm_desc* d) {
    if (!d) return fail(NOP_E_INVALID, "descriptor is NULL");
    if (d->abi_version != NOP_ABI_VERSION) return fail(NOP_E_INVALID, "ABI version mismatch");
    if (d->dtype < NOP_DTYPE_FP32 || d->dtype > NOP_DTYPE_FP16) return fail(NOP_E_INVALID, "unknown dtype");
    if (d->batch < 0 || d->points < 0 || d->channels < 1)
        return fail(NOP_E_INVALID, "batch and points must be >= 0 and channels >= 1");
    if (d->channels > kMaxChannels) return fail(NOP_E_UNSUPPORTED, "more than 8192 channels");
    if (!(d->eps >= 0.f)) return fail(NOP_E_INVALID, "eps must be a number >= 0");
    if (d->points && d->batch > (int64_t)0x7fffffffffLL / d->points / d->channels)
        return fail(NOP_E_UNSUPPORTED, "a field of more than 2^39 values");
    return NOP_OK;
}

template <class T, int V, int NC>
int32_t launch_fwd(const Args& a, const Cut& c, bool residual, bool q8, cudaStream_t s) {
    const unsigned grid = (unsigned)ceil_div(c.tiles, c.warps / c.W);
    const int smem = (q8 ? 2 : 1) * c.warps * 32 * V * 4;
    const int threads = c.warps * 32;
    if (q8) {
        if (residual) k_fwd<T, V, NC, true, true><<<grid, threads, smem, s>>>(a);
        else k_fwd<T, V, NC, false, true><<<grid, threads, smem, s>>>(a);
    } else {
        if (residual) k_fwd<T, V, NC, true, false><<<grid, threads, smem, s>>>(a);
        else k_fwd<T, V, NC, false, false><<<grid, threads, smem, s>>>(a);
    }
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

template <class T, int V, int NC>
int32_t launch_bwd(const Args& a, const Cut& c, unsigned grid, int dev, cudaStream_t s) {
    const int smem = (4 * c.warps * 32 * V + (NC ? 0 : a.C)) * 4;
    const int threads = c.warps * 32;
    if (smem > 48 * 1024) {  // (with the sums of many channels)
        constexpr int most = (4 * kMaxWarps * 32 * V + kMaxChannels) * 4;
        const int32_t rc = a.gr ? allow_smem<k_bwd<T, V, NC, true>>(dev, most) : allow_smem<k_bwd<T, V, NC, false>>(dev, most);
        if (rc != NOP_OK) return rc;
    }
    if (a.gr) k_bwd<T, V, NC, true><<<grid, threads, smem, s>>>(a);
    else k_bwd<T, V, NC, false><<<grid, threads, smem, s>>>(a);
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

// f(T{}, V, NC) for the call's type and cut (as compile-time constants); fp32 has no 8-value vectors, the
// backward (at most 16 / 2 bytes a load) neither
template <bool BWD, class F>
int32_t dispatch(int dtype, const Cut& c, F&& f) {
    auto by_nc = [&](auto t, auto v) {
        switch (c.NC) {
            case 8: return f(t, v, std::integral_constant<int, 8>{});
            case 16: return f(t, v, std::integral_constant<int, 16>{});
            default: return f(t, v, std::integral_constant<int, 0>{});
        }
    };
    auto by_v = [&](auto t) {
        constexpr bool wide = sizeof(t) == 2;
        switch (c.V) {
            case 8:
                if constexpr (wide && !BWD) return by_nc(t, std::integral_constant<int, 8>{});
                break;
            case 4:
                if constexpr (wide || !BWD) return by_nc(t, std::integral_constant<int, 4>{});
                break;
            case 2: return by_nc(t, std::integral_constant<int, 2>{});
            default: break;
        }
        return by_nc(t, std::integral_constant<int, 1>{});
    };
    if (dtype == NOP_DTYPE_FP32) return by_v(float{});
    if (dtype == NOP_DTYPE_BF16) return by_v(__nv_bfloat16{});
    return by_v(__half{});
}

// every pointer on a 16-byte boundary (wide loads), or at least on its type's
bool on_16(std::initializer_list<const void*> ps) {
    uintptr_t all = 0;
    for (const void* p : ps) all |= (uintptr_t)p;
    return all % 16 == 0;
}

}  // namespace rms
}  // namespace nop

using namespace nop;

extern "C" {

int32_t nop_rms_norm_forward(const nop_norm_desc* d, const void* x, const void* residual, const float* weight, void* y,
                             void* r, void* q, float* scale, void* stream) {
    int32_t rc = rms::check(d);
    if (rc != NOP_OK) return rc;
    if (d->batch == 0 || d->points == 0) return NOP_OK;
    const bool q8 = q != nullptr;
    if (!x || (!q8 && !y) || (q8 && !scale)) return fail(NOP_E_INVALID, "x and y (or q and scale) must be non-NULL");
    if (q8 && y) return fail(NOP_E_INVALID, "either y or q is written");
    if ((residual == nullptr) != (r == nullptr))
        return fail(NOP_E_INVALID, "residual and r must be given together");
    const int size = d->dtype == NOP_DTYPE_FP32 ? 4 : 2;
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y | (uintptr_t)r) % size || (uintptr_t)scale % 4 ||
        (uintptr_t)weight % 4)
        return fail(NOP_E_ALIGNMENT, "a pointer is not aligned to its type");
    int dev = 0, sms = 148;
    if ((rc = current_device(&dev, &sms)) != NOP_OK) return rc;
    const rms::Cut c = rms::cut_of(*d, size, rms::on_16({x, residual, y, r, q}), sms, false);
    if (ceil_div(c.tiles, c.warps / c.W) > 0x7fffffffLL) return fail(NOP_E_UNSUPPORTED, "too many points");
    rms::Args a{};
    a.x = x;
    a.res = residual;
    a.w = weight;
    a.y = y;
    a.r = r;
    a.q = static_cast<uint8_t*>(q);
    a.scale = scale;
    a.C = d->channels;
    a.W = c.W;
    a.P = d->points;
    a.groups = c.groups;
    a.tiles = c.tiles;
    a.eps = d->eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return rms::dispatch<false>(d->dtype, c, [&](auto t, auto v, auto nc) {
        return rms::launch_fwd<decltype(t), decltype(v)::value, decltype(nc)::value>(a, c, residual != nullptr, q8, s);
    });
}

int32_t nop_rms_norm_backward_workspace_size(const nop_norm_desc* d, size_t* bytes) {
    const int32_t rc = rms::check(d);
    if (rc != NOP_OK) return rc;
    if (!bytes) return fail(NOP_E_INVALID, "bytes is NULL");
    const rms::Cut c = rms::cut_of(*d, 4, false, 1, true);
    *bytes = (size_t)d->channels * c.max_grid(rms::kMaxSms) * (c.warps / c.W) * sizeof(float);
    return NOP_OK;
}

int32_t nop_rms_norm_backward(const nop_norm_desc* d, const void* r, const float* weight, const void* gy, const void* gr,
                              void* gx, float* gw, void* workspace, size_t workspace_bytes, void* stream) {
    int32_t rc = rms::check(d);
    if (rc != NOP_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->batch == 0 || d->points == 0) {
        if (gw) NOP_CUDA_TRY(cudaMemsetAsync(gw, 0, d->channels * sizeof(float), s));
        return NOP_OK;
    }
    if (!r || !gy) return fail(NOP_E_INVALID, "r and gy must be non-NULL");
    if (!gx && !gw) return NOP_OK;
    const int size = d->dtype == NOP_DTYPE_FP32 ? 4 : 2;
    if (((uintptr_t)r | (uintptr_t)gy | (uintptr_t)gr | (uintptr_t)gx) % size || (uintptr_t)gw % 4 ||
        (uintptr_t)weight % 4 || (uintptr_t)workspace % 4)
        return fail(NOP_E_ALIGNMENT, "a pointer is not aligned to its type");
    int dev = 0, sms = 148;
    if ((rc = current_device(&dev, &sms)) != NOP_OK) return rc;
    const rms::Cut c = rms::cut_of(*d, size, rms::on_16({r, gy, gr, gx}), sms, true);
    const int slots = c.warps / c.W;
    int64_t grid = ceil_div(c.tiles, slots);
    if (grid > c.max_grid(sms)) grid = c.max_grid(sms);
    const int64_t rows = grid * slots;
    if (gw && (!workspace || workspace_bytes < (size_t)rows * d->channels * sizeof(float)))
        return fail(NOP_E_WORKSPACE, "workspace missing or too small");
    rms::Args a{};
    a.x = r;
    a.gy = gy;
    a.gr = gr;
    a.gx = gx;
    a.w = weight;
    a.partial = gw ? static_cast<float*>(workspace) : nullptr;
    a.C = d->channels;
    a.W = c.W;
    a.P = d->points;
    a.groups = c.groups;
    a.tiles = c.tiles;
    a.eps = d->eps;
    rc = rms::dispatch<true>(d->dtype, c, [&](auto t, auto v, auto nc) {
        return rms::launch_bwd<decltype(t), decltype(v)::value, decltype(nc)::value>(a, c, (unsigned)grid, dev, s);
    });
    if (rc != NOP_OK || !gw) return rc;
    rms::k_reduce<<<d->channels, 128, 0, s>>>(a.partial, (int)rows, gw);
    NOP_CUDA_TRY(cudaGetLastError());
    return NOP_OK;
}

}  // extern "C"
