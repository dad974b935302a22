// The paged cache in 8 bits, as its kernels share it.
//
// A layer's keys (and values) are e4m3 numbers [page][kv head][slot][dim] and a float32 scale per (page, kv head): the
// number that a byte stands for is e4m3 * scale.  A scale is a power of two 2^e, -48 <= e <= 48.  So a row that is stored
// again under a larger scale loses nothing above e4m3's subnormals, scores take a page's scale in one exact
// multiplication, and the attention kernels may carry a value page's scale as an integer in the exponent of a weight.
// The range leaves float32 room for what is multiplied with it: weights times 2^(-e) stay finite and, between any two
// pages, above 2^-126 unless they differ by 2^30 besides.
//
// Every e4m3 number is a float16 number: the attention kernels hand keys and values to the tensor cores as float16, exactly,
// with one conversion per two numbers, and float32 accumulators.
//
// A key row that holds NaN marks a token whose key or value was not finite when it was stored; its values are stored as
// zeros.  Value rows therefore never hold NaN, and a weight of 0 removes a masked token whatever it held.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>
#include <utility>

namespace {

constexpr int Q8_E_MIN = -48, Q8_E_MAX = 48;

// 2^e for the exponents that scales have (and sums of a few)
__device__ __forceinline__ float q8_pow2(int e) { return __int_as_float((e + 127) << 23); }
// the exponent of a scale as stored: of the power of two at or below it, within the range (0 is 2^-48, an infinity or NaN 2^48), by every
// kernel, so that scales which the append did not leave mean the same to all of them
__device__ __forceinline__ int q8_exponent(float scale) {
    return min(max(((__float_as_int(scale) >> 23) & 0xff) - 127, Q8_E_MIN), Q8_E_MAX);
}

// the smallest e in [-48, 48] with m <= 448 * 2^e, from the bits of m >= 0: 448 = 1.75 * 2^8, so a mantissa above
// 1.75 (0x600000) carries into the exponent
__device__ __forceinline__ int q8_exponent_for(int bits) {
    if (bits == 0) return Q8_E_MIN;
    const int e = ((bits + 0x1fffff) >> 23) - 127 - 8;
    return min(max(e, Q8_E_MIN), Q8_E_MAX);
}

// two e4m3 numbers (the low byte first) as two float16
__device__ __forceinline__ uint32_t q8_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n.reg .b16 l;\ncvt.u16.u32 l, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(two));
    return r;
}
// four e4m3 numbers as two pairs of float16
__device__ __forceinline__ void q8_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
// Loads of what the kernel does not write that stay where they are written: the compiler moves plain ones down to their
// use, past the work that they were to overlap with.
__device__ __forceinline__ int load_early(const int* p) {
    int v;
    asm volatile("ld.global.nc.b32 %0, [%1];\n" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float load_early(const float* p) {
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];\n" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float4 load_early(const float4* p) {
    float4 v;
    asm volatile("ld.global.nc.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_early(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// the nearest e4m3 numbers, ties to even; beyond +-448 they stay at it, NaN is NaN
__device__ __forceinline__ uint32_t q8_pack2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t q8_half2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// ---- what the attention kernels share ----

constexpr float kMoveAt = 7.875f;           // the reference moves when the maximum has grown by more than 2^7.875
constexpr float kLift = 7.f;                // weights are carried 2^7 up: float16's range below 1
// What is above this moves the reference m.  Rounded down: where float32 numbers are 2, 4 or 8 apart, m - 7 may be m - 8, and with the
// maximum at m + 8 a weight would be 2^16, which is no float16 number; it is at most m + 6 so.
__device__ __forceinline__ float moves_above(float m) { return __fadd_rd(m, kMoveAt); }
constexpr float kLog2e = 1.4426950408889634f;

// 2^x, the hardware approximation: 2^-22 off at most, far below half a step of what the weight is rounded to or summed with
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// The power of two that brings a row's largest magnitude m (its bits) to 2^14 <= m < 2^15, as an exponent; the other way
// round it is in the row's factor.  Rows of zeros and of tiny numbers stop at 2^100.
__device__ __forceinline__ int row_shift(int bits) { return min(14 + 127 - (bits >> 23), 100); }

// What a part with reference m and sum l counts beside the reference of all parts.  A part without a seen key has -inf and 0;
// one that met only NaN has -inf and NaN, which stays.
__device__ __forceinline__ float part_factor(float m, float l, float all) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - all);
}
__device__ __forceinline__ void add_scaled(float4& x, float f, const float4& y) {
    x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
}
// x / l, zeros where no key was seen
template <typename T> __device__ __forceinline__ void store_row4(T* dst, const float4& x, float l) {
    const float4 y = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x / l, x.y / l, x.z / l, x.w / l);
    if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<float4*>(dst) = y;
    }
}

// The tile'th of the tiles of `per` rows into which the requests' portions, rows q_start[s] .. q_start[s + 1], are cut.  Where the
// requests are no more than lanes, their portions come one after another in the order of their contexts' ends, the longest
// last (kernels start with the last tile: what takes long begins first), else as they stand.
struct Portion {
    int req, tok0, end, pos0;            // request, the tile's first row, the portion's end, the first row's position
};
// By a whole warp, a request a lane (400 requests of 2 tokens behind 100: 101 us, with a walk by one thread 322).  False: there are
// fewer tiles.
__device__ __forceinline__ bool find_portion(const int* q_start, const int* start_pos, int n_requests, int per, int tile, Portion& p) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < n_requests; s0 += 32) {
        const int s = s0 + lane;
        const bool there = s < n_requests;
        const int begin = there ? max(q_start[s], 0) : 0, end = there ? q_start[s + 1] : 0, start = there ? start_pos[s] : 0;
        const int rows = end - begin, mine = rows > 0 ? (rows + per - 1) / per : 0;
        int upto = mine;                                     // tiles up to the lane's last
        if (n_requests <= 32) {
            upto = 0;
            const int ctx = start + rows;
            for (int j = 0; j < n_requests; j++) {
                const int other = __shfl_sync(0xffffffffu, ctx, j), tiles = __shfl_sync(0xffffffffu, mine, j);
                if (other < ctx || (other == ctx && j <= lane)) upto += tiles;
            }
        } else {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int before = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += before;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < upto && tile >= upto - mine);
        if (hit) {
            const int l = __ffs(hit) - 1, into = (tile - (upto - mine)) * per;
            p.req = s0 + l;
            p.tok0 = __shfl_sync(0xffffffffu, begin + into, l);
            p.end = __shfl_sync(0xffffffffu, end, l);
            p.pos0 = __shfl_sync(0xffffffffu, start + into, l);
            return true;
        }
        tile -= __reduce_add_sync(0xffffffffu, mine);
    }
    return false;
}

// The end of the keys that a table of max_blocks pages can name, at most hi: a position behind the table costs no walk there.  A few
// tiles below 2^31, so that the places of the tiles that are looked up ahead are numbers too.
__device__ __forceinline__ int keys_end(int64_t hi, int max_blocks, int page_size) {
    const int64_t table = (int64_t)max_blocks * page_size, end = table < 0x7ffff000 ? table : 0x7ffff000;
    return (int)(hi < end ? hi : end);
}

// Joins the ranges of a row (token, head) in order, HD / 4 threads a row.  What bounds it is the chain of its loads, so the first
// parts are on their way before the references are known, and whether the row is any request's is asked at the store only (rows
// of tokens outside [q_start[0], q_start[n_requests]) are left alone; q_start NULL: all are joined).  512 tokens of 32 heads of 128 in two
// parts by themselves: 9 us (a CTA a row that asked first: 20).
template <int HD> constexpr int q8_join_rows = 256 / (HD / 4);
template <typename T, int HD>
__global__ void __launch_bounds__(q8_join_rows<HD> * (HD / 4))
q8_join_kernel(T* __restrict__ out, const float* __restrict__ part_o, const float* __restrict__ part_ml, int ranges, int n_heads,
               int64_t n_rows, const int* __restrict__ q_start, int n_requests) {
    constexpr int AHEAD = 4;
    griddep_wait();
    griddep_launch();
    const int64_t at = (int64_t)blockIdx.x * q8_join_rows<HD> + threadIdx.x / (HD / 4);
    if (at >= n_rows) return;
    const int d = threadIdx.x % (HD / 4) * 4;
    const float2* ml = reinterpret_cast<const float2*>(part_ml) + at * ranges;
    const float4* part = reinterpret_cast<const float4*>(part_o + at * ranges * HD + d);
    float4 ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (i < ranges) ahead[i] = load_early(part + i * (HD / 4));
    const int from = q_start ? q_start[0] : 0, to = q_start ? q_start[n_requests] : 0;
    float m = -INFINITY;
#pragma unroll 4
    for (int r = 0; r < ranges; r++) m = fmaxf(m, ml[r].x);
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (i < ranges) {
            const float f = part_factor(ml[i].x, ml[i].y, m);
            l += f * ml[i].y;
            add_scaled(x, f, ahead[i]);
        }
#pragma unroll 4
    for (int r = AHEAD; r < ranges; r++) {
        const float f = part_factor(ml[r].x, ml[r].y, m);
        l += f * ml[r].y;
        add_scaled(x, f, part[r * (HD / 4)]);
    }
    const int token = (int)(at / n_heads);
    if (!q_start || (token >= from && token < to)) store_row4(out + at * HD + d, x, l);
}
template <typename T, int HD>
void launch_join(void* out, const float* part_o, const float* part_ml, int ranges, int n_heads, int64_t n_rows, const int* q_start,
                 int n_requests, cudaStream_t stream) {
    kllm_launch((q8_join_kernel<T, HD>), dim3((unsigned)((n_rows + q8_join_rows<HD> - 1) / q8_join_rows<HD>)), dim3(q8_join_rows<HD> * (HD / 4)), 0,
                stream, (T*)out, part_o, part_ml, ranges, n_heads, n_rows, q_start, n_requests);
}

// Calls an entry point with its arguments from a block of 8-byte numbers, one each: addresses and integers as int64, floating-point
// numbers as double.  A caller in Python packs such a block in a fraction of the time that as many typed arguments take.
template <typename T> T packed_argument(const int64_t* p) {
    if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>((uintptr_t)*p);
    else if constexpr (std::is_floating_point_v<T>) { double x; memcpy(&x, p, 8); return (T)x; }
    else return (T)*p;
}
template <typename... A, size_t... I> int call_packed(int (*entry)(A...), const int64_t* args, std::index_sequence<I...>) {
    return entry(packed_argument<A>(args + I)...);
}
template <typename... A> [[maybe_unused]] int call_packed(int (*entry)(A...), const void* args) {
    return call_packed(entry, (const int64_t*)args, std::index_sequence_for<A...>());
}

// Once per device: more than 48 KB of dynamic shared memory for a kernel.
[[maybe_unused]] cudaError_t open_shared_memory(const void* kernel, int bytes, std::atomic<uint64_t>& opened) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (opened.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) opened.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace
