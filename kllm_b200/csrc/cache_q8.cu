// Rotary encoding of a step's queries and keys, and the write of keys and values into the paged cache in 8 bits
// (q8.cuh: e4m3 numbers, one power of two per page and kv head).
//
// For a page that a step writes to, with the rows x_r that it stores there and the exponent e_old of the rows that the
// page holds already (none if the step writes its first slot):
//     e = max(e_old, the smallest e' with max |x_r| <= 448 * 2^e'),   byte = e4m3(x_r * 2^-e),
// and where e > e_old the earlier rows become e4m3(old * 2^(e_old - e)).  A row whose key or value is not finite counts
// for no maximum; its key is stored as NaN and its value as 0.
// The rotation is that of rope.cu: rotate_half, float32, angles from a table computed in float64.  A key is rounded once,
// from the rotated float32 numbers to e4m3.
//
// One CTA takes (a few tokens, one kv head): it rotates the query heads of that kv head's group for its tokens, and stores
// whole runs of rows: the first token of a request's rows in a page (the request's first token of the step, or slot 0)
// does it for all of them, so that exactly one CTA touches a (page, kv head) and its scale.  Each run is read twice, the
// second time from the first-level cache: once for the rows' largest magnitudes (integer maxima in shared memory: the order does
// not matter), once to store.
#include "q8.cuh"

KLLM_EXPORT_LAST_ERROR(cache_q8)

namespace {

constexpr int kThreads = 128;
constexpr int kMaxPage = 4096;              // two words of shared memory per row of a run

template <typename T, int U> __device__ __forceinline__ void load(const T* p, float (&v)[U]) {
    if constexpr (U == 1) {
        v[0] = to_f32(*p);
    } else if constexpr (sizeof(T) == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
}
template <typename T, int U> __device__ __forceinline__ void store(T* p, const float (&v)[U]) {
    if constexpr (U == 1) {
        *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 2) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        uint2 w;
        w.x = *reinterpret_cast<uint32_t*>(&a); w.y = *reinterpret_cast<uint32_t*>(&b);
        *reinterpret_cast<uint2*>(p) = w;
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
}
template <int U> __device__ __forceinline__ void store8(uint8_t* p, const float (&v)[U], float mul) {
    if constexpr (U == 1) *p = (uint8_t)(q8_pack2(v[0] * mul, 0.f) & 0xff);
    else *reinterpret_cast<uint32_t*>(p) = q8_pack2(v[0] * mul, v[1] * mul) | (q8_pack2(v[2] * mul, v[3] * mul) << 16);
}
template <int U> __device__ __forceinline__ void fill8(uint8_t* p, uint32_t byte) {
    if constexpr (U == 1) *p = (uint8_t)byte;
    else *reinterpret_cast<uint32_t*>(p) = byte * 0x01010101u;
}
template <int U> __device__ __forceinline__ int largest(const float (&v)[U]) {
    int m = 0;
#pragma unroll
    for (int i = 0; i < U; i++) m = max(m, __float_as_int(v[i]) & 0x7fffffff);
    return m;
}

// a[], b[]: U numbers of a row at j and U at j + half, turned by the angles of the row's position
template <typename T, int U>
__device__ __forceinline__ void turn(const T* row, const float* cs, int j, int half, float (&a)[U], float (&b)[U]) {
    float c[U], s[U], x[U], y[U];
    load<T, U>(row + j, x);
    load<T, U>(row + j + half, y);
    load<float, U>(cs + j, c);
    load<float, U>(cs + half + j, s);
#pragma unroll
    for (int i = 0; i < U; i++) {
        a[i] = x[i] * c[i] - y[i] * s[i];
        b[i] = y[i] * c[i] + x[i] * s[i];
    }
}

// U numbers at a time: 4 where half the rotary width, strides and addresses allow it, else 1
template <typename T, int U>
__global__ void __launch_bounds__(kThreads)
rope_append_q8_kernel(T* q_out, int64_t qo_stride, const T* q, int64_t q_stride, const T* __restrict__ k,
                      int64_t k_stride, const T* __restrict__ v, int64_t v_stride, const float* __restrict__ cos_sin, int n_pos,
                      const int* __restrict__ positions, const int* __restrict__ token_req, const int* __restrict__ q_start,
                      int n_requests, const int* __restrict__ block_table, int max_blocks, uint8_t* __restrict__ kcache,
                      uint8_t* __restrict__ vcache, float* __restrict__ kscale, float* __restrict__ vscale, int n_pages,
                      int n_tokens, int group, int n_kv, int hd, int rot, int page_size, int chunk) {
    extern __shared__ int row_max[];          // [2][rows of the run]: the largest magnitude's bits of keys, of values
    __shared__ int s_max[2];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, g = blockIdx.y;
    const int n_all = min(n_tokens, q_start[n_requests]);          // rows behind the last request are left alone
    const int t0 = blockIdx.x * chunk, t1 = min(n_all, t0 + chunk);
    const int half = rot >> 1;
    const int pairs = half / U, tail = (hd - rot) / U;             // units of a row

    // queries of this kv head's group
    const int per_head = pairs + (q_out != q ? tail : 0);
    if (per_head > 0) {
        for (int u = tid; u < (t1 - t0) * group * per_head; u += kThreads) {
            const int i = u % per_head, th = u / per_head;
            const int t = t0 + th / group, h = g * group + th % group;
            const int p = positions[t];
            const T* src = q + (int64_t)t * q_stride + (int64_t)h * hd;
            T* dst = q_out + (int64_t)t * qo_stride + (int64_t)h * hd;
            if (i < pairs) {
                if (p < 0 || p >= n_pos) continue;
                float a[U], b[U];
                turn<T, U>(src, cos_sin + (int64_t)p * rot, i * U, half, a, b);
                store<T, U>(dst + i * U, a);
                store<T, U>(dst + half + i * U, b);
            } else {
                float a[U];
                load<T, U>(src + rot + (i - pairs) * U, a);
                store<T, U>(dst + rot + (i - pairs) * U, a);
            }
        }
    }

    // runs of rows that begin among these tokens
    for (int t = t0; t < t1; t++) {
        const int req = token_req ? token_req[t] : t;
        if (req < 0 || req >= n_requests) continue;
        const int p = positions[t], begin = q_start[req], end = min(q_start[req + 1], n_all);
        if (p < 0 || (rot > 0 && p >= n_pos)) continue;
        const int lp = p / page_size, slot = p - lp * page_size;
        if ((slot != 0 && t != begin) || lp >= max_blocks) continue;
        const int page = block_table[(int64_t)req * max_blocks + lp];
        if (page < 0 || page >= n_pages) continue;
        int rows = min(end - t, page_size - slot);
        if (rot > 0) rows = min(rows, n_pos - p);
        if (rows <= 0) continue;
        int* kmax = row_max;
        int* vmax = row_max + rows;
        const int64_t cell = (int64_t)page * n_kv + g;
        // read before the meetings below: thread 0 stores the new scales behind them
        const int ke_old = slot ? q8_exponent(kscale[cell]) : Q8_E_MIN, ve_old = slot ? q8_exponent(vscale[cell]) : Q8_E_MIN;
        __syncthreads();                                          // the run before is done with the maxima
        for (int r = tid; r < 2 * rows; r += kThreads) row_max[r] = 0;
        if (tid < 2) s_max[tid] = 0;
        __syncthreads();
        const int k_units = pairs + tail, v_units = hd / U, units = k_units + v_units;
        const T* k0 = k + (int64_t)t * k_stride + (int64_t)g * hd;
        const T* v0 = v + (int64_t)t * v_stride + (int64_t)g * hd;
        const float* cs0 = cos_sin + (int64_t)p * rot;
        for (int u = tid; u < rows * units; u += kThreads) {
            const int r = u / units, i = u - r * units;
            float a[U];
            if (i < pairs) {
                float b[U];
                turn<T, U>(k0 + r * k_stride, cs0 + (int64_t)r * rot, i * U, half, a, b);
                atomicMax(&kmax[r], max(largest<U>(a), largest<U>(b)));
            } else if (i < k_units) {
                load<T, U>(k0 + r * k_stride + rot + (i - pairs) * U, a);
                atomicMax(&kmax[r], largest<U>(a));
            } else {
                load<T, U>(v0 + r * v_stride + (i - k_units) * U, a);
                atomicMax(&vmax[r], largest<U>(a));
            }
        }
        __syncthreads();
        for (int r = tid; r < rows; r += kThreads) {
            const int a = kmax[r], b = vmax[r];
            if (max(a, b) >= 0x7f800000) kmax[r] = -1;            // an infinity or NaN in the key or the value
            else { atomicMax(&s_max[0], a); atomicMax(&s_max[1], b); }
        }
        __syncthreads();
        const int ke = max(ke_old, q8_exponent_for(s_max[0])), ve = max(ve_old, q8_exponent_for(s_max[1]));
        uint8_t* kp = kcache + cell * page_size * hd;
        uint8_t* vp = vcache + cell * page_size * hd;
        // rows that the page holds already
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const int e = w ? ve : ke, e_old = w ? ve_old : ke_old;
            if (!slot || e == e_old) continue;
            uint32_t* c = reinterpret_cast<uint32_t*>(w ? vp : kp);
            const float mul = q8_pow2(max(e_old - e, -126));
            for (int u = tid; u < slot * hd / 4; u += kThreads) {
                const uint32_t x = c[u];
                const uint32_t lo = q8_to_f16x2(x & 0xffffu), hi = q8_to_f16x2(x >> 16);
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                c[u] = q8_pack2(a.x * mul, a.y * mul) | (q8_pack2(b.x * mul, b.y * mul) << 16);
            }
        }
        // the new rows
        const float kmul = q8_pow2(-ke), vmul = q8_pow2(-ve);
        kp += (int64_t)slot * hd;
        vp += (int64_t)slot * hd;
        for (int u = tid; u < rows * units; u += kThreads) {
            const int r = u / units, i = u - r * units;
            const bool bad = kmax[r] < 0;
            float a[U];
            if (i < pairs) {
                uint8_t* dst = kp + (int64_t)r * hd + i * U;
                if (bad) {
                    fill8<U>(dst, 0x7f);
                    fill8<U>(dst + half, 0x7f);
                } else {
                    float b[U];
                    turn<T, U>(k0 + r * k_stride, cs0 + (int64_t)r * rot, i * U, half, a, b);
                    store8<U>(dst, a, kmul);
                    store8<U>(dst + half, b, kmul);
                }
            } else if (i < k_units) {
                const int d = rot + (i - pairs) * U;
                if (bad) {
                    fill8<U>(kp + (int64_t)r * hd + d, 0x7f);
                } else {
                    load<T, U>(k0 + r * k_stride + d, a);
                    store8<U>(kp + (int64_t)r * hd + d, a, kmul);
                }
            } else {
                const int d = (i - k_units) * U;
                if (bad) {
                    fill8<U>(vp + (int64_t)r * hd + d, 0);
                } else {
                    load<T, U>(v0 + r * v_stride + d, a);
                    store8<U>(vp + (int64_t)r * hd + d, a, vmul);
                }
            }
        }
        if (tid == 0) {
            kscale[cell] = q8_pow2(ke);
            vscale[cell] = q8_pow2(ve);
        }
    }
}

template <typename T, int U, typename... A>
void launch(dim3 grid, size_t smem, cudaStream_t s, A... a) {
    kllm_launch((rope_append_q8_kernel<T, U>), grid, dim3(kThreads), smem, s, a...);
}

}  // namespace

// q_out [n, heads*hd] at qo_stride (may be q itself), q/k/v rows dense at their strides, element type dtype; cos_sin float32
// [n_pos, rot] (rot 0: no rotation); token_req may be NULL (token t is request t's only one); caches [pages, n_kv, page, hd]
// e4m3, scales float32 [pages, n_kv].  Nothing is read or stored for a token whose position is negative, outside the
// table of angles, or without a page.
extern "C" int kllm_rope_append_q8(void* q_out, int64_t qo_stride, const void* q, int64_t q_stride, const void* k,
                                   int64_t k_stride, const void* v, int64_t v_stride, const float* cos_sin, int n_pos,
                                   const int* positions, const int* token_req, const int* q_start, int n_requests,
                                   const int* block_table, int max_blocks, void* kcache, void* vcache, float* kscale,
                                   float* vscale, int n_pages, int n_tokens, int n_heads, int n_kv, int hd, int rot,
                                   int page_size, int dtype, void* stream) {
    if (n_tokens <= 0 || n_requests <= 0) return 0;
    if (n_kv <= 0 || n_heads <= 0 || n_heads % n_kv) KLLM_FAIL("append (8 bits): %d heads over %d kv heads", n_heads, n_kv);
    if (hd <= 0 || hd % 32 || hd > 256) KLLM_FAIL("append (8 bits): head size %d is not a multiple of 32 up to 256", hd);
    if (rot < 0 || rot % 2 || rot > hd) KLLM_FAIL("append (8 bits): rotary width %d of a head of %d", rot, hd);
    if (page_size <= 0 || page_size > kMaxPage) KLLM_FAIL("append (8 bits): page size %d, at most %d", page_size, kMaxPage);
    if (n_kv > 65535) KLLM_FAIL("append (8 bits): %d kv heads, at most 65535", n_kv);
    if (dtype != KLLM_F32 && dtype != KLLM_BF16) KLLM_FAIL("append (8 bits): element type %d", dtype);
    const int es = dtype == KLLM_F32 ? 4 : 2;
    // one CTA a token where every request brings one, else 16 tokens a CTA
    const int chunk = n_tokens <= n_requests ? 1 : 16;
    const dim3 grid((n_tokens + chunk - 1) / chunk, n_kv);
    const size_t smem = (size_t)2 * 4 * (page_size < n_tokens ? page_size : n_tokens);
    const bool four = rot % 8 == 0 && !((qo_stride | q_stride | k_stride | v_stride) & 3) &&
                      !(((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & (4 * es - 1)) &&
                      !((uintptr_t)cos_sin & 15) && !(((uintptr_t)kcache | (uintptr_t)vcache) & 3);
    if (((uintptr_t)kcache | (uintptr_t)vcache) & 3) KLLM_FAIL("append (8 bits): the caches must be 4-byte aligned");
    const cudaStream_t s = (cudaStream_t)stream;
#define KLLM_GO(T, U)                                                                                                        \
    launch<T, U>(grid, smem, s, (T*)q_out, qo_stride, (const T*)q, q_stride, (const T*)k, k_stride, (const T*)v, v_stride,  \
                 cos_sin, n_pos, positions, token_req, q_start, n_requests, block_table, max_blocks, (uint8_t*)kcache,      \
                 (uint8_t*)vcache, kscale, vscale, n_pages, n_tokens, n_heads / n_kv, n_kv, hd, rot, page_size, chunk)
    if (dtype == KLLM_F32) {
        if (four) KLLM_GO(float, 4); else KLLM_GO(float, 1);
    } else {
        if (four) KLLM_GO(bf16, 4); else KLLM_GO(bf16, 1);
    }
#undef KLLM_GO
    KLLM_LAUNCH_STATUS();
}
