// Rotary encoding of a step's queries and keys, and the write of keys and values into the paged cache in 8 bits
// (q8.cuh: e4m3 numbers, one power of two per page and kv head).
//
// For a page that a step writes to, with the rows x_r that it stores there and the exponent e_old of the rows that the
// page holds already (none if the step writes its first slot):
//     e = max(e_old, the smallest e' with max |x_r| <= 448 * 2^e'),   byte = e4m3(x_r * 2^-e),
// and where e > e_old the earlier rows become e4m3(old * 2^(e_old - e)).  A row whose key or value is not finite counts
// for no maximum; its key is stored as NaN and its value as 0.
// The rotation is that of rope.cu: rotate_half, float32, angles from a table computed in float64.  A key's byte is the e4m3
// number next to its exact rotation by the table's angles, and its page's scale follows the exact rotation too.
//
// What bounds it: bytes, and for few tokens a chain of dependent loads.  A CTA takes a few tokens and one of two jobs: it
// rotates some of their query heads, or it stores whole runs of rows of some kv heads: the first token of a request's rows in a
// page (the request's first token of the step, or slot 0) does it for all of them, so that exactly one CTA touches a (page,
// kv head) and its scale.  A thread keeps its place in the rows and walks the rows, without a division per unit.  A run is
// read twice, the second time from the first-level cache: once for the largest magnitudes (integer maxima in shared memory:
// their order does not matter), once to store.  Rows that are not finite are rare, as are maxima beside a border of the scales: the former
// are marked on the first way, and only where there are any of either the maxima are taken again, without those rows and from the exact
// rotation.
//
// Measured, back to back: 8 tokens of 32 + 2 * 4 heads of 64 in bfloat16 3.6 us, 2048 tokens 9.5 us (20 MB, 2.2 TB/s; copies at
// 6.45 TB/s would take 3.2); 3842 tokens in float32 of 32 + 2 * 32 heads of 128 in 9 portions on pages of 16 76.3 us (285 MB, 3.7 TB/s,
// 58 % of a copy), in bfloat16 63.0.  These wait for their loads (6 of 12 cycles between two instructions of a warp, issue slots 57 % busy) at the 32
// warps an SM that 64 registers leave.  A run's numbers kept in registers between the two ways, and more loads in flight at more registers, were both slower.
// Rounding the exact rotation costs 8 to 13 % of that: rounded from float32 arithmetic one number in a million was its neighbour.
#include "q8.cuh"

KLLM_EXPORT_LAST_ERROR(cache_q8)

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16;                  // tokens a CTA looks after
template <int U> constexpr int kBatch = U == 8 ? 2 : 4;   // query heads whose numbers a thread requests together
constexpr int kMaxHeads = 4;                // kv heads a CTA stores at most
constexpr int kMaxRunBytes = 65536;         // what a CTA reads of a run, where several kv heads are more
constexpr int kMaxMarks = 32768;            // rows of a run x kv heads: a byte each
constexpr int kMaxPage = 4096;

template <typename T, int U> __device__ __forceinline__ void load(const T* p, float (&v)[U]) {
    if constexpr (U == 1) {
        v[0] = to_f32(*p);
    } else if constexpr (U == 8 && sizeof(T) == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t h[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(h[i] << 16); v[2 * i + 1] = __uint_as_float(h[i] & 0xffff0000u); }
    } else if constexpr (U == 8) {
        const float4 w = *reinterpret_cast<const float4*>(p), x = *reinterpret_cast<const float4*>(p + 4);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        v[4] = x.x; v[5] = x.y; v[6] = x.z; v[7] = x.w;
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
    } else if constexpr (U == 8) {
        static_assert(sizeof(T) == 2, "16 bytes");
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            h[i] = *reinterpret_cast<const uint32_t*>(&a);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    } else if constexpr (sizeof(T) == 2) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        uint2 w;
        w.x = *reinterpret_cast<uint32_t*>(&a); w.y = *reinterpret_cast<uint32_t*>(&b);
        *reinterpret_cast<uint2*>(p) = w;
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
}
// U numbers times mul as e4m3, four a word
template <int U> constexpr int kWords = (U + 3) / 4;
template <int U> __device__ __forceinline__ void pack8(const float* v, float mul, uint32_t (&w)[kWords<U>]) {
    if constexpr (U == 1) {
        w[0] = q8_pack2(v[0] * mul, 0.f) & 0xff;
    } else {
#pragma unroll
        for (int i = 0; i < U / 4; i++)
            w[i] = q8_pack2(v[4 * i] * mul, v[4 * i + 1] * mul) | (q8_pack2(v[4 * i + 2] * mul, v[4 * i + 3] * mul) << 16);
    }
}
template <int U> __device__ __forceinline__ void store8(uint8_t* p, const uint32_t (&w)[kWords<U>]) {
    if constexpr (U == 1) *p = (uint8_t)w[0];
    else if constexpr (U == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}
template <int U> __device__ __forceinline__ void fill8(uint8_t* p, uint32_t byte) {
    if constexpr (U == 1) *p = (uint8_t)byte;
    else if constexpr (U == 8) *reinterpret_cast<uint2*>(p) = make_uint2(byte * 0x01010101u, byte * 0x01010101u);
    else *reinterpret_cast<uint32_t*>(p) = byte * 0x01010101u;
}

// A unit of a row is 2 U numbers: v[0 .. U) from place `at`, v[U .. 2U) from `at2`.  Units below `pairs` are the two halves of
// U rotated pairs, the others 2 U neighbours.
struct Unit {
    int at, at2;
};
template <int U> __device__ __forceinline__ Unit unit_of(int i, int pairs, int half, int rot) {
    if (i < pairs) return Unit{i * U, i * U + half};
    const int at = rot + (i - pairs) * 2 * U;
    return Unit{at, at + U};
}
struct Run {                                // rows of one request in one page that this step stores
    int token, page, slot, rows;
};
template <typename T, int U> struct Raw {   // a unit as it is read, with its angles
    float x[U], y[U], c[U], s[U];
};
template <typename T, int U> __device__ __forceinline__ void read_unit(Raw<T, U>& w, const T* row, Unit u, bool turned, const float* cs, int half) {
    load<T, U>(row + u.at, w.x);
    load<T, U>(row + u.at2, w.y);
    if (turned) {
        load<float, U>(cs + u.at, w.c);
        load<float, U>(cs + half + u.at, w.s);
    }
}
template <typename T, int U> __device__ __forceinline__ void turn(const Raw<T, U>& w, bool turned, float (&v)[2 * U]) {
#pragma unroll
    for (int i = 0; i < U; i++) {
        v[i] = turned ? w.x[i] * w.c[i] - w.y[i] * w.s[i] : w.x[i];
        v[U + i] = turned ? w.y[i] * w.c[i] + w.x[i] * w.s[i] : w.y[i];
    }
}

// a c - b s with its last bit set where it is not exact and cut towards zero ("to odd"): a further rounding to fewer bits gives what
// rounding the exact number once gives.  The products' and the sum's errors are exact float32 numbers (fma; two-sum), their sum is off by
// 2^-46 of the products.
__device__ __noinline__ float turned_to_odd(float a, float c, float b, float s) {
    const float p = a * c, n = -b * s;
    const float ep = fmaf(a, c, -p), en = fmaf(-b, s, -n);
    const float r = __fadd_rn(p, n), t = __fsub_rn(r, p);
    const float e = __fadd_rn(__fadd_rn(__fsub_rn(p, __fsub_rn(r, t)), __fsub_rn(n, t)), __fadd_rn(ep, en));
    const float sum = __fadd_rn(r, e), u = __fsub_rn(sum, r);
    const float rest = __fadd_rn(__fsub_rn(r, __fsub_rn(sum, u)), __fsub_rn(e, u));
    if (!(fabsf(sum) < INFINITY)) return r;
    int bits = __float_as_int(sum);
    if (rest != 0.f) {
        if (bits << 1 && (rest < 0.f) != (sum < 0.f)) bits--;
        bits |= 1;
    }
    return __int_as_float(bits);
}
template <typename T, int U> __device__ __forceinline__ void turn_to_odd(const Raw<T, U>& w, float (&v)[2 * U]) {
#pragma unroll
    for (int i = 0; i < U; i++) {
        v[i] = turned_to_odd(w.x[i], w.c[i], w.y[i], w.s[i]);
        v[U + i] = turned_to_odd(w.y[i], w.c[i], -w.x[i], w.s[i]);
    }
}
// Whether a largest magnitude (its bits) is so near to a border of the scales, 448 * 2^e, that the exact one may be beyond it: a pair
// turned in float32 arithmetic by angles on a circle is off by 1.5 last places of its larger number.
__device__ __forceinline__ bool beside_border(int bits) { return (unsigned)((bits & 0x7fffff) - 0x5ffffc) <= 8u; }
// The unit as e4m3.  Turned numbers are within 1.5 last places here (the error of the product that is rounded first is taken off the
// sum): where a number times 1 - 2^-21 and times 1 + 2^-21 round alike, so does the exact one.  A unit with one that does not
// (once in 10^4 units) is taken again.
template <typename T, int U>
__device__ __forceinline__ void pack_unit(const Raw<T, U>& w, bool turned, float mul, uint32_t (&a)[kWords<U>], uint32_t (&b)[kWords<U>]) {
    float v[2 * U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        v[i] = w.x[i]; v[U + i] = w.y[i];
        if (turned) {
            const float p = __fmul_rn(w.y[i], w.s[i]), q = __fmul_rn(w.x[i], w.s[i]);
            v[i] = __fsub_rn(fmaf(w.x[i], w.c[i], -p), fmaf(w.y[i], w.s[i], -p));
            v[U + i] = __fadd_rn(fmaf(w.y[i], w.c[i], q), fmaf(w.x[i], w.s[i], -q));
        }
    }
    const float wide = turned ? mul * 0x1p-21f : 0.f;
    uint32_t a2[kWords<U>], b2[kWords<U>];
    pack8<U>(v, mul - wide, a); pack8<U>(v, mul + wide, a2);
    pack8<U>(v + U, mul - wide, b); pack8<U>(v + U, mul + wide, b2);
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < kWords<U>; i++) differ |= (a[i] ^ a2[i]) | (b[i] ^ b2[i]);
    if (differ) {
        turn_to_odd<T, U>(w, v);
        pack8<U>(v, mul, a);
        pack8<U>(v + U, mul, b);
    }
}

// U = 8 (bfloat16) or 4 where half the rotary width, strides and addresses allow it, else 1: what a thread reads at a time is 16 bytes
template <typename T, int U>
__global__ void __launch_bounds__(kThreads, 4)
rope_append_q8_kernel(T* q_out, int64_t qo_stride, const T* q, int64_t q_stride, const T* __restrict__ k,
                      int64_t k_stride, const T* __restrict__ v, int64_t v_stride, const float* __restrict__ cos_sin, int n_pos,
                      const int* __restrict__ positions, const int* __restrict__ token_req, const int* __restrict__ q_start,
                      int n_requests, const int* __restrict__ block_table, int max_blocks, uint8_t* __restrict__ kcache,
                      uint8_t* __restrict__ vcache, float* __restrict__ kscale, float* __restrict__ vscale, int n_pages,
                      int n_tokens, int n_heads, int q_heads, int n_kv, int kv_heads, int hd, int rot, int page_size, int chunk) {
    extern __shared__ uint8_t bad[];          // [rows of the run][kv heads]: an infinity or NaN in the key or the value
    __shared__ int s_max[kMaxHeads][2], s_pos[kChunk], s_req[kChunk], s_runs, s_any;
    __shared__ Run s_run[kChunk];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, threads = blockDim.x, kv_ctas = (n_kv + kv_heads - 1) / kv_heads;
    const int n_all = min(n_tokens, q_start[n_requests]);          // rows behind the last request are left alone
    const int t0 = blockIdx.x * chunk, t1 = min(n_all, t0 + chunk);
    if (t0 >= t1) return;
    if (tid < t1 - t0) {
        s_pos[tid] = positions[t0 + tid];
        s_req[tid] = token_req ? token_req[t0 + tid] : t0 + tid;
    }
    const int half = rot >> 1, pairs = half / U, per_row = hd / (2 * U);     // units of a row
    __syncthreads();

    if ((int)blockIdx.y >= kv_ctas) {
        // queries: a CTA's share of the heads, in place only the pairs.  A thread keeps (token, place in the head), for which it
        // reads the angles once, and walks the heads.
        const int per_head = q_out != q ? per_row : pairs, h0 = ((int)blockIdx.y - kv_ctas) * q_heads, h1 = min(h0 + q_heads, n_heads);
        const int places = chunk * per_head, together = max(1, threads / places);        // heads at a time
        for (int c0 = 0; c0 < places; c0 += threads) {
            const int first = places <= threads ? tid / places : 0, c = places <= threads ? tid - first * places : c0 + tid;
            const int t = c / per_head, i = c - t * per_head;
            if (first >= together || t >= t1 - t0) continue;
            const Unit unit = unit_of<U>(i, pairs, half, rot);
            const bool turned = i < pairs;
            const int p = s_pos[t];
            if (turned && (p < 0 || p >= n_pos)) continue;
            Raw<T, U> w;
            if (turned) {
                load<float, U>(cos_sin + (int64_t)p * rot + unit.at, w.c);
                load<float, U>(cos_sin + (int64_t)p * rot + half + unit.at, w.s);
            }
            const T* src = q + (int64_t)(t0 + t) * q_stride;
            T* dst = q_out + (int64_t)(t0 + t) * qo_stride;
            for (int h = h0 + first; h < h1; h += kBatch<U> * together) {
                float x[kBatch<U>][U], y[kBatch<U>][U];
#pragma unroll
                for (int j = 0; j < kBatch<U>; j++)
                    if (h + j * together < h1) {
                        load<T, U>(src + (int64_t)(h + j * together) * hd + unit.at, x[j]);
                        load<T, U>(src + (int64_t)(h + j * together) * hd + unit.at2, y[j]);
                    }
#pragma unroll
                for (int j = 0; j < kBatch<U>; j++)
                    if (h + j * together < h1) {
                        float z[2 * U];
#pragma unroll
                        for (int l = 0; l < U; l++) { w.x[l] = x[j][l]; w.y[l] = y[j][l]; }
                        turn<T, U>(w, turned, z);
                        T* to = dst + (int64_t)(h + j * together) * hd;
                        store<T, U>(to + unit.at, *reinterpret_cast<const float(*)[U]>(z));
                        store<T, U>(to + unit.at2, *reinterpret_cast<const float(*)[U]>(z + U));
                    }
            }
        }
        return;
    }

    const int g0 = blockIdx.y * kv_heads, heads = min(kv_heads, n_kv - g0);
    const int units = 2 * per_row, cols = heads * units;            // a head's key, then its value
    const int together = threads / cols, first = tid / cols, col = tid - first * cols, h = col / units, i = col - h * units;
    const bool key = i < per_row, turned = i < pairs, mine = first < together;
    const Unit unit = key ? unit_of<U>(i, pairs, half, rot) : unit_of<U>(i - per_row, 0, 0, 0);
    const T* src = (key ? k : v) + (int64_t)(g0 + h) * hd;
    const int64_t src_stride = key ? k_stride : v_stride;
    // runs of rows that begin among these tokens: found by a thread per token
    if (tid < 32) {
        int page = -1, slot = 0, rows = 0;
        if (tid < t1 - t0) {
            const int req = s_req[tid], p = s_pos[tid], t = t0 + tid;
            if (req >= 0 && req < n_requests && p >= 0 && (rot == 0 || p < n_pos)) {
                const int lp = p / page_size, begin = q_start[req], end = min(q_start[req + 1], n_all);
                slot = p - lp * page_size;
                if ((slot == 0 || t == begin) && lp < max_blocks) page = block_table[(int64_t)req * max_blocks + lp];
                rows = min(end - t, page_size - slot);
                if (rot > 0) rows = min(rows, n_pos - p);
            }
        }
        const bool run = page >= 0 && page < n_pages && rows > 0;
        const unsigned runs = __ballot_sync(0xffffffffu, run);
        if (run) s_run[__popc(runs & ((1u << tid) - 1))] = Run{tid, page, slot, rows};
        if (tid == 0) s_runs = __popc(runs);
    }
    __syncthreads();
    for (int n = 0; n < s_runs; n++) {
        const int t = t0 + s_run[n].token, p = s_pos[s_run[n].token], page = s_run[n].page, slot = s_run[n].slot, rows = s_run[n].rows;
        const int64_t cell0 = (int64_t)page * n_kv + g0, cell = cell0 + h;
        // read before the meetings below: the new scales are stored behind them
        const int ke_old = slot ? q8_exponent(kscale[cell]) : Q8_E_MIN, ve_old = slot ? q8_exponent(vscale[cell]) : Q8_E_MIN;
        const T* row0 = src + (int64_t)t * src_stride;
        const float* cs0 = cos_sin + (int64_t)p * rot;
        auto read = [&](int r, Raw<T, U>& w) {
            read_unit<T, U>(w, row0 + (int64_t)r * src_stride, unit, turned, cs0 + (int64_t)r * rot, half);
        };
        __syncthreads();                                            // the run before is done with the marks and the maxima
        for (int j = tid; j < rows * heads; j += threads) bad[j] = 0;
        if (tid < 2 * kMaxHeads) s_max[tid >> 1][tid & 1] = 0;
        if (tid == 0) s_any = 0;
        __syncthreads();
        int m = 0;
#pragma unroll (U == 8 ? 2 : 4)
        for (int r = first; mine && r < rows; r += together) {
            Raw<T, U> w;
            float x[2 * U];
            read(r, w);
            turn<T, U>(w, turned, x);
            int mr = 0;
#pragma unroll
            for (int j = 0; j < 2 * U; j++) mr = max(mr, __float_as_int(x[j]) & 0x7fffffff);
            if (mr >= 0x7f800000) { bad[r * heads + h] = 1; s_any = 1; }
            else m = max(m, mr);
        }
        if (mine) atomicMax(&s_max[h][key], m);
        __syncthreads();
        const bool any = s_any != 0;
        bool again = any;
        for (int j = 0; j < heads; j++) again = again || (rot > 0 && beside_border(s_max[j][1]));
        if (again) {                                                // the same for all threads: without those rows, from the exact rotation
            __syncthreads();
            if (tid < 2 * kMaxHeads) s_max[tid >> 1][tid & 1] = 0;
            __syncthreads();
            m = 0;
            for (int r = first; mine && r < rows; r += together) {
                if (bad[r * heads + h]) continue;
                Raw<T, U> w;
                float x[2 * U];
                read(r, w);
                turn<T, U>(w, false, x);
                if (turned) turn_to_odd<T, U>(w, x);
#pragma unroll
                for (int j = 0; j < 2 * U; j++) m = max(m, __float_as_int(x[j]) & 0x7fffffff);
            }
            if (mine) atomicMax(&s_max[h][key], m);
            __syncthreads();
        }
        const int ke = max(ke_old, q8_exponent_for(s_max[h][1])), ve = max(ve_old, q8_exponent_for(s_max[h][0]));
        uint8_t* page_rows = (key ? kcache : vcache) + cell * page_size * hd;
        const int e = key ? ke : ve, e_old = key ? ke_old : ve_old;
        // rows that the page holds already
        if (mine && slot && e != e_old) {
            const float down = q8_pow2(e_old - e);
            for (int r = first; r < slot; r += together) {
                uint8_t* at[2] = {page_rows + (int64_t)r * hd + unit.at, page_rows + (int64_t)r * hd + unit.at2};
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if constexpr (U == 1) {
                        const uint32_t lo = q8_to_f16x2(*at[j]);
                        *at[j] = (uint8_t)(q8_pack2(__half22float2(*reinterpret_cast<const __half2*>(&lo)).x * down, 0.f) & 0xff);
                    } else {
#pragma unroll
                        for (int l = 0; l < U; l += 4) {
                            uint32_t* p4 = reinterpret_cast<uint32_t*>(at[j] + l);
                            uint32_t lo, hi;
                            q8_to_f16x4(*p4, lo, hi);
                            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                            *p4 = q8_pack2(a.x * down, a.y * down) | (q8_pack2(b.x * down, b.y * down) << 16);
                        }
                    }
                }
            }
        }
        // the new rows
        const float mul = q8_pow2(-e);
#pragma unroll (U == 8 ? 2 : 4)
        for (int r = first; mine && r < rows; r += together) {
            uint8_t* dst = page_rows + (int64_t)(slot + r) * hd;
            if (any && bad[r * heads + h]) {
                fill8<U>(dst + unit.at, key ? 0x7f : 0);
                fill8<U>(dst + unit.at2, key ? 0x7f : 0);
                continue;
            }
            Raw<T, U> w;
            read(r, w);
            uint32_t lower[kWords<U>], upper[kWords<U>];
            pack_unit<T, U>(w, turned, mul, lower, upper);
            store8<U>(dst + unit.at, lower);
            store8<U>(dst + unit.at2, upper);
        }
        if (first == 0 && i == 0) {
            kscale[cell] = q8_pow2(ke);
            vscale[cell] = q8_pow2(ve);
        }
    }
}

template <typename T, int U, typename... A>
void launch(dim3 grid, int threads, size_t smem, cudaStream_t s, A... a) {
    kllm_launch((rope_append_q8_kernel<T, U>), grid, dim3(threads), smem, s, a...);
}

}  // namespace

// q_out [n, heads*hd] at qo_stride (may be q itself), q/k/v rows dense at their strides, element type dtype; cos_sin float32
// [n_pos, rot] (rot 0: no rotation); token_req may be NULL (token t is request t's only one); caches [pages, n_kv, page, hd]
// e4m3, scales float32 [pages, n_kv].  Nothing is stored in the caches for a token whose position is negative or outside the table of
// angles, or that has no page.  Its query: of a position outside the table only what is not rotated is written, and that only where
// q_out is not q; a query of a token without a page is rotated and written like any other.
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
    // Eight numbers at a time cost registers (spills) that calls of a few microseconds notice and larger ones do not: 8 tokens of 32 + 2 * 4 heads
    // of 64 4.3 us against 3.8 with four, 3000 of 24 + 2 * 8 of 96 (12 M numbers) 19.8 against 18.7, 3842 of 32 + 2 * 8 of 128 (24 M) 28.5 against
    // 29.0, of 32 + 2 * 32 (47 M) 63.7 against 71.7.
    const bool many = (int64_t)n_tokens * (n_heads + 2 * n_kv) * hd >= 1 << 24;
    const bool eight = many && dtype == KLLM_BF16 && rot % 16 == 0 && !((qo_stride | q_stride | k_stride | v_stride) & 7) &&
                       !(((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos_sin) & 15) &&
                       !(((uintptr_t)kcache | (uintptr_t)vcache) & 7);
    const bool four = rot % 8 == 0 && !((qo_stride | q_stride | k_stride | v_stride) & 3) &&
                      !(((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & (4 * es - 1)) &&
                      !((uintptr_t)cos_sin & 15) && !(((uintptr_t)kcache | (uintptr_t)vcache) & 3);
    // A CTA a token where every request brings one, else one for sixteen.  kv heads a CTA: as many as its threads cover, at most
    // four, as long as there are runs enough for two CTAs on each of the 148 SMs and the run stays in the first-level cache beside those of the SM's
    // other CTAs until it is read again.  Microseconds for 3842 tokens in 9 portions with 1, 2, 4, 8 heads of 128 a CTA: float32, 32 kv
    // heads, pages of 16 (16 KB a head) 88, 73, 70, 79, pages of 64 76, 77, 81, 119; bfloat16 (four numbers at a time), 8 kv heads, pages of 16
    // 34, 29, 27, 31; 4 x 2048 tokens, pages of 64 69, 64, 68, 68.
    const int chunk = n_tokens <= n_requests ? 1 : kChunk;
    const int units = eight ? hd / 8 : four ? hd / 4 : hd;      // of a head's key and value
    const int run = page_size < n_tokens ? page_size : n_tokens;
    const int64_t runs = chunk == 1 ? n_tokens : (int64_t)n_tokens / page_size + n_requests;
    int kv_heads = kThreads / units < kMaxHeads ? kThreads / units : kMaxHeads;
    if (kv_heads > runs * n_kv / 296) kv_heads = (int)(runs * n_kv / 296);
    if (kv_heads > kMaxMarks / run) kv_heads = kMaxMarks / run;
    const int64_t head_bytes = (int64_t)(chunk == 1 ? 1 : run) * 2 * hd * es;
    if (kv_heads > kMaxRunBytes / head_bytes) kv_heads = (int)(kMaxRunBytes / head_bytes);
    if (kv_heads < 1) kv_heads = 1;
    if (kv_heads > n_kv) kv_heads = n_kv;
    // threads for the longest run
    int threads = 64;
    while (threads < kv_heads * units || (threads < kThreads && threads < (chunk == 1 ? 1 : run) * kv_heads * units)) threads *= 2;
    // query heads a CTA: a batch for every thread, as long as that leaves two CTAs an SM
    const int chunks = (n_tokens + chunk - 1) / chunk;
    int q_heads = (eight ? kBatch<8> : kBatch<4>) * (threads / (chunk * (units / 2)) > 0 ? threads / (chunk * (units / 2)) : 1);
    while (q_heads > 1 && (int64_t)chunks * ((n_heads + q_heads - 1) / q_heads) < 296) q_heads /= 2;
    const int kv_ctas = (n_kv + kv_heads - 1) / kv_heads, q_ctas = rot > 0 || q_out != q ? (n_heads + q_heads - 1) / q_heads : 0;
    if (kv_ctas + q_ctas > 65535) KLLM_FAIL("append (8 bits): %d heads over %d kv heads", n_heads, n_kv);
    const dim3 grid(chunks, kv_ctas + q_ctas);
    const size_t smem = (size_t)run * kv_heads;
    if (((uintptr_t)kcache | (uintptr_t)vcache) & 3) KLLM_FAIL("append (8 bits): the caches must be 4-byte aligned");
    const cudaStream_t s = (cudaStream_t)stream;
#define KLLM_GO(T, U)                                                                                                        \
    launch<T, U>(grid, threads, smem, s, (T*)q_out, qo_stride, (const T*)q, q_stride, (const T*)k, k_stride, (const T*)v, v_stride,  \
                 cos_sin, n_pos, positions, token_req, q_start, n_requests, block_table, max_blocks, (uint8_t*)kcache,      \
                 (uint8_t*)vcache, kscale, vscale, n_pages, n_tokens, n_heads, q_heads, n_kv, kv_heads, hd, rot, page_size, chunk)
    if (dtype == KLLM_F32) {
        if (four) KLLM_GO(float, 4); else KLLM_GO(float, 1);
    } else {
        if (eight) KLLM_GO(bf16, 8); else if (four) KLLM_GO(bf16, 4); else KLLM_GO(bf16, 1);
    }
#undef KLLM_GO
    KLLM_LAUNCH_STATUS();
}
extern "C" int kllm_rope_append_q8_packed(const void* args) { return call_packed(&kllm_rope_append_q8, args); }
