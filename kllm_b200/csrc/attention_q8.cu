// Causal grouped-query attention over the paged cache in 8 bits (q8.cuh), one library per head size (-DKLLM_HD, a multiple
// of 32 up to 256).  Queries and outputs are bfloat16 or float32.
//
// For a row (the token at position p, head h over kv head g) and the keys j it sees, max(0, p + 1 - window) <= j <= p:
//     s_j = log2(e) scale (q . k8_j) 2^ek(j),      weight 2^s_j / sum,      out = sum_j weight_j v8_j 2^ev(j)
// where ek, ev are the exponents of the page's scales.  A value page's exponent goes into the weight's: with a reference M,
//     w_j = 2^(s_j + ev(j) - M + 7),   l = sum_j w_j 2^-ev(j),   O = sum_j w_j v8_j,   out = O / l,
// so that one exponential a score serves both sums, whatever the pages' scales are.  The reference follows the running
// maximum of s_j + ev(j) and is moved only when that has grown by more than 8: w stays below 2^15, a float16 number, and
// what is smaller than 2^-32 of the largest weight is lost.
//
// Products run on the tensor cores in float16 with float32 sums (mma.sync m16n8k16): e4m3 numbers are float16 numbers.
// A row of bfloat16 queries is one float16 operand, exactly, after division by a power of two that brings its largest
// magnitude to 2^14..2^15; a float32 row is the sum of three (33 bits).  Weights are one float16 (11 bits: half a step is
// 2^-12, against bfloat16's 2^-9), beside float32 queries two (22 bits).  A row with an infinity or NaN among its queries
// becomes NaN.
//
// Keys without a page (a table entry outside the pages, a place behind the table's end) are not seen.  A row that sees no
// key becomes zeros.
#include "q8.cuh"

#ifndef KLLM_HD
#error "compile with -DKLLM_HD=<head size, a multiple of 32 up to 256>"
#endif

KLLM_EXPORT_LAST_ERROR(attention_q8)

namespace {

constexpr int HD = KLLM_HD;
static_assert(HD % 32 == 0 && HD >= 32 && HD <= 256, "head sizes: multiples of 32 up to 256");
constexpr float kMoveAt = 8.f;              // the reference moves when the maximum has grown by 2^8
constexpr float kLift = 7.f;                // weights are carried 2^7 up: float16's range below 1
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Parts { static constexpr int Q = 1, P = 1; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 2; };

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// 2^x, the hardware approximation: 2^-22 off at most, far below half a step of what the weight is rounded to or summed with
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// The power of two that brings a row's largest magnitude m (its bits) to 2^14 <= m < 2^15, as an exponent; the other way
// round it is in the row's factor.  Rows of zeros and of tiny numbers stop at 2^100.
__device__ __forceinline__ int row_shift(int bits) { return min(14 + 127 - (bits >> 23), 100); }

// part i of x: x = p0 + p1 + p2 + ..., each a float16 number
template <int N> __device__ __forceinline__ void split(float x, __half (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        p[i] = __float2half_rn(x);
        x -= __half2float(p[i]);
    }
}

// ---- single tokens ---------------------------------------------------------------------------------------------------
//
// What bounds it: bytes.  Every warp walks its own tiles of keys with no shared memory and no meeting: a lane's loads of a
// key tile are the tensor core's operand itself.  Keys are the M side (A, 16 keys x 16 dims), the heads of the group the N
// side (8 at a time): lane (g, t) = (lane / 4, lane % 4) holds rows g and g + 8, and because the order of the dims under a
// sum is free, its dims are 16 neighbours of every 64 (one 16-byte load), the same for the queries.  The second product
// takes values as A with the dims as M: lane (g, t) holds HD / 8 neighbouring dims of keys 2t, 2t + 1, 2t + 8, 2t + 9, two
// keys' bytes are interleaved (prmt) and converted to the pairs that the operand wants, and the weights, whose layout
// is (key, head), become the B operand by an 8 x 8 transposition in registers (movmatrix).  A tile's keys are loaded while
// the values before them are used, a tile's values while its scores are computed.

constexpr int DEC_KT = HD <= 128 ? 32 : 16;              // keys of a warp's tile
constexpr int DEC_MT = DEC_KT / 16;
constexpr int DEC_WARPS = 4;
constexpr int KW = HD % 64 == 0 ? 4 : 2;                 // words of a lane's piece of a key row
constexpr int KC = HD / (16 * KW);                       // pieces of a key row (16 * KW dims each)
constexpr int VW = HD / 32;                              // words of a lane's piece of a value row

template <typename T, int NG> struct DecodeShape {
    static constexpr int NQ = Parts<T>::Q;
    static constexpr int QREGS = HD / 16 * 2 * NQ * NG;
    static constexpr bool Q_IN_REGS = QREGS <= 32;
    // CTAs an SM: what the registers of a lane allow without spills
    static constexpr int CTAS = HD <= 64 ? (NG == 1 ? 5 : 4) : HD <= 128 ? (NG == 1 ? 4 : 3) : 2;
};

struct DecodeArgs {
    void* out;
    float* part_o;               // [n, heads, ranges, HD], part_ml [n, heads, ranges, 2]: NULL with one range
    float* part_ml;
    const void* q;
    int64_t q_stride;
    const uint8_t* kcache;
    const uint8_t* vcache;
    const float* kscale;
    const float* vscale;
    const int* positions;
    const int* token_req;
    const int* block_table;
    int max_blocks, n_pages, n_requests, n_heads, n_kv, subs, heads_per_cta, page_size, window, ranges;
    float scale;
};

template <int W> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&r)[W]) {
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + 4 * i));
            r[i] = v.x; r[i + 1] = v.y; r[i + 2] = v.z; r[i + 3] = v.w;
        }
    } else if constexpr (W % 2 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + 4 * i));
            r[i] = v.x; r[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; i++) r[i] = __ldg(reinterpret_cast<const uint32_t*>(p + 4 * i));
    }
}

__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
__device__ __forceinline__ float peer_load(const float* p, unsigned rank) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p), b;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(b) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(b));
    return v;
}

// grid: (ranges * cluster, kv heads * subgroups of heads, tokens), clusters along x; a cluster's CTAs take neighbouring
// parts of a range and join through distributed shared memory
template <typename T, int NG>
__global__ void __launch_bounds__(DEC_WARPS * 32, (DecodeShape<T, NG>::CTAS))
attn_decode_q8_kernel(const DecodeArgs a) {
    constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P, NH = 8 * NG;
    constexpr bool Q_IN_REGS = DecodeShape<T, NG>::Q_IN_REGS;
    constexpr int QSM = HD / 16 * NQ * NG * 32;                       // uint2 per lane: [kk][part][ng][lane]
    extern __shared__ __align__(16) unsigned char smem[];
    uint2* sq = reinterpret_cast<uint2*>(smem);                       // the queries as operands
    float* so = reinterpret_cast<float*>(smem + QSM * 8);             // [warps][NH][HD], then the CTA's sum [NH][HD]
    __shared__ float s_ml[DEC_WARPS][NH][2];                          // references and sums of the warps
    __shared__ float s_cta[NH][2];                                    // ... of the CTA
    __shared__ float s_factor[NH];                                    // log2(e) scale 2^(the row's power), NaN: the row is
    __shared__ int s_amax[NH];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int token = blockIdx.z, kvh = blockIdx.y / a.subs, sub = blockIdx.y % a.subs;
    const int head0 = kvh * (a.n_heads / a.n_kv) + sub * a.heads_per_cta, nh = a.heads_per_cta;
    const int req = a.token_req ? a.token_req[token] : token;
    const int p = (req >= 0 && req < a.n_requests) ? a.positions[token] : -1;
    const int hi = p + 1, lo = (a.window > 0 && hi > a.window) ? hi - a.window : 0;

    // queries: largest magnitude per head, then the operand's words
    const T* q = (const T*)a.q + (int64_t)token * a.q_stride + (int64_t)head0 * HD;
    if (tid < NH) s_amax[tid] = 0;
    __syncthreads();
    for (int h = warp; h < nh; h += DEC_WARPS) {
        int m = 0;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) m = max(m, __float_as_int(to_f32(q[h * HD + i * 32 + lane])) & 0x7fffffff);
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) s_amax[h] = m;
    }
    __syncthreads();
    if (tid < NH) s_factor[tid] = s_amax[tid] >= 0x7f800000 ? __int_as_float(0x7fffffff)
                                                            : a.scale * kLog2e * q8_pow2(-row_shift(s_amax[tid]));
    for (int u = tid; u < HD / 16 * NG * 32; u += DEC_WARPS * 32) {
        const int l = u & 31, ng = (u >> 5) % NG, kk = (u >> 5) / NG;
        const int h = ng * 8 + (l >> 2), t = l & 3;
        // dims of the step's k = 2t, 2t + 1 and 2t + 8, 2t + 9: four neighbours of lane t's piece
        const int d = (kk / KW) * (16 * KW) + t * (4 * KW) + (kk % KW) * 4;
        __half parts[4][NQ];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x = 0.f;
            if (h < nh && s_amax[h] < 0x7f800000) x = to_f32(q[h * HD + d + i]) * q8_pow2(row_shift(s_amax[h]));
            split<NQ>(x, parts[i]);
        }
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            const __half2 w0 = __halves2half2(parts[0][j], parts[1][j]), w1 = __halves2half2(parts[2][j], parts[3][j]);
            sq[((kk * NQ + j) * NG + ng) * 32 + l] = make_uint2(*reinterpret_cast<const uint32_t*>(&w0), *reinterpret_cast<const uint32_t*>(&w1));
        }
    }
    __syncthreads();
    uint2 qr[Q_IN_REGS ? HD / 16 * NQ * NG : 1];
    if constexpr (Q_IN_REGS) {
#pragma unroll
        for (int i = 0; i < HD / 16 * NQ * NG; i++) qr[i] = sq[i * 32 + lane];
    }
    float factor[NG][2], m_ref[NG][2], l_run[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ng++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            factor[ng][i] = s_factor[ng * 8 + 2 * t4 + i];
            m_ref[ng][i] = -INFINITY;
            l_run[ng][i] = 0.f;
        }

    // this warp's tiles: the token's tiles [first, last) in one part per CTA, a part's tiles in turn over the warps
    const int parts = gridDim.x, part = blockIdx.x;
    const int first = lo / DEC_KT, last = (hi + DEC_KT - 1) / DEC_KT;      // tiles start at multiples of their size
    const int per = (last - first + parts - 1) / parts;
    const int tile_lo = first + part * per, tile_hi = min(last, tile_lo + per);

    const int* table = a.block_table + (int64_t)(req < 0 ? 0 : req) * a.max_blocks;
    // what a lane knows of key tile * DEC_KT + lane % DEC_KT: its row in the stores (-1: not seen), its scales' exponents
    auto lookup = [&](int tile, int& row, float& kmul, int& ev) {
        row = -1; kmul = 0.f; ev = 0;
        const int key = tile * DEC_KT + (lane & (DEC_KT - 1));
        if (tile >= tile_hi || key < lo || key >= hi) return;
        const int lp = key / a.page_size;
        if (lp >= a.max_blocks) return;
        const int page = __ldg(table + lp);
        if ((unsigned)page >= (unsigned)a.n_pages) return;
        const int cell = page * a.n_kv + kvh;
        row = cell * a.page_size + key - lp * a.page_size;
        kmul = __ldg(a.kscale + cell);
        ev = q8_exponent(__ldg(a.vscale + cell));
    };
    uint32_t kr[DEC_MT][2][KC][KW], vr[DEC_MT][4][VW];
    auto load_k = [&](int row) {
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = max(__shfl_sync(0xffffffffu, row, mt * 16 + i * 8 + g8), 0);
                const uint8_t* src = a.kcache + (int64_t)r * HD + t4 * (4 * KW);
#pragma unroll
                for (int c = 0; c < KC; c++) load_words<KW>(src + c * (16 * KW), kr[mt][i][c]);
            }
    };
    auto load_v = [&](int row) {
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = __shfl_sync(0xffffffffu, row, mt * 16 + (i >> 1) * 8 + 2 * t4 + (i & 1));
                load_words<VW>(a.vcache + (int64_t)max(r, 0) * HD + g8 * (HD / 8), vr[mt][i]);
                if (r < 0) {                         // what is not seen may hold anything, NaN too
#pragma unroll
                    for (int w = 0; w < VW; w++) vr[mt][i][w] = 0;
                }
            }
    };
    float o[HD / 16][NG][4];
#pragma unroll
    for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int ng = 0; ng < NG; ng++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][ng][j] = 0.f;

    int row, row_next, ev, ev_next;
    float kmul, kmul_next;
    int tile = tile_lo + warp;
    lookup(tile, row, kmul, ev);
    if (tile < tile_hi) { load_k(row); load_v(row); }
    for (; tile < tile_hi; tile += DEC_WARPS) {
        const bool more = tile + DEC_WARPS < tile_hi;
        lookup(tile + DEC_WARPS, row_next, kmul_next, ev_next);
        float s[DEC_MT][NG][4];
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[mt][ng][j] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int w = 0; w < KW; w++) {
                const int kk = c * KW + w;
#pragma unroll
                for (int j = NQ - 1; j >= 0; j--)                   // the smallest part first
#pragma unroll
                    for (int ng = 0; ng < NG; ng++) {
                        const int at = (kk * NQ + j) * NG + ng;
                        const uint2 b = Q_IN_REGS ? qr[Q_IN_REGS ? at : 0] : sq[at * 32 + lane];
#pragma unroll
                        for (int mt = 0; mt < DEC_MT; mt++)
                            mma16816(s[mt][ng], q8_to_f16x2(kr[mt][0][c][w] & 0xffffu), q8_to_f16x2(kr[mt][1][c][w] & 0xffffu),
                                     q8_to_f16x2(kr[mt][0][c][w] >> 16), q8_to_f16x2(kr[mt][1][c][w] >> 16), b.x, b.y);
                    }
            }
        if (more) load_k(row_next);
        // scores, in units of log2, with the values' exponents
        bool grown = false;
        float inv[DEC_MT][2];                       // 2^-ev of the lane's keys g8 and g8 + 8
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int src = mt * 16 + i * 8 + g8;
                const int r = __shfl_sync(0xffffffffu, row, src);
                const float km = __shfl_sync(0xffffffffu, kmul, src);
                const int e = __shfl_sync(0xffffffffu, ev, src);
                inv[mt][i] = q8_pow2(-e);
#pragma unroll
                for (int ng = 0; ng < NG; ng++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float& x = s[mt][ng][2 * i + j];
                        x = r < 0 ? -INFINITY : fmaf(x * km, factor[ng][j], (float)e);
                        grown = grown || x > m_ref[ng][j] + kMoveAt;
                    }
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int mt = 0; mt < DEC_MT; mt++) mx = fmaxf(mx, fmaxf(s[mt][ng][j], s[mt][ng][2 + j]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    if (mx > m_ref[ng][j] + kMoveAt) {              // the same for every lane of the head
                        const float corr = m_ref[ng][j] == -INFINITY ? 0.f : exp2f(m_ref[ng][j] - mx);
                        m_ref[ng][j] = mx;
                        l_run[ng][j] *= corr;
#pragma unroll
                        for (int i = 0; i < HD / 16; i++) {
                            o[i][ng][j] *= corr;
                            o[i][ng][2 + j] *= corr;
                        }
                    }
                }
        }
        uint32_t pb[DEC_MT][NP][NG][2];
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float w[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float ref = m_ref[ng][j] == -INFINITY ? 0.f : m_ref[ng][j] - kLift;
                        w[j] = fast_exp2(s[mt][ng][2 * i + j] - ref);
                        l_run[ng][j] = fmaf(w[j], inv[mt][i], l_run[ng][j]);
                    }
                    __half h0[NP], h1[NP];
                    split<NP>(w[0], h0);
                    split<NP>(w[1], h1);
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        const __half2 hh = __halves2half2(h0[k], h1[k]);
                        pb[mt][k][ng][i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hh));
                    }
                }
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int w = 0; w < VW; w++)
#pragma unroll
                for (int half = 0; half < 2; half++) {              // dims 4w, 4w + 1, then 4w + 2, 4w + 3
                    const unsigned sel = half ? 0x7362u : 0x5140u;
                    const uint32_t x = __byte_perm(vr[mt][0][w], vr[mt][1][w], sel), y = __byte_perm(vr[mt][2][w], vr[mt][3][w], sel);
                    const uint32_t a0 = q8_to_f16x2(x & 0xffffu), a1 = q8_to_f16x2(x >> 16);
                    const uint32_t a2 = q8_to_f16x2(y & 0xffffu), a3 = q8_to_f16x2(y >> 16);
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--)
#pragma unroll
                        for (int ng = 0; ng < NG; ng++) mma16816(o[2 * w + half][ng], a0, a1, a2, a3, pb[mt][k][ng][0], pb[mt][k][ng][1]);
                }
        if (more) load_v(row_next);
        row = row_next; kmul = kmul_next; ev = ev_next;
    }

    // join: the warps of the CTA in order, then the CTAs of the cluster in order
#pragma unroll
    for (int ng = 0; ng < NG; ng++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l_run[ng][j] += __shfl_xor_sync(0xffffffffu, l_run[ng][j], d);
            const int h = ng * 8 + 2 * t4 + j;
            if (g8 == 0) { s_ml[warp][h][0] = m_ref[ng][j]; s_ml[warp][h][1] = l_run[ng][j]; }
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
                // dims of rows g and g + 8 of step i: neighbours g * HD / 8 + 2 i, + 1
                float2 v = make_float2(o[i][ng][j], o[i][ng][2 + j]);
                *reinterpret_cast<float2*>(so + ((warp * NH + h) * HD + g8 * (HD / 8) + 2 * i)) = v;
            }
        }
    __syncthreads();
    for (int u = tid; u < nh * HD; u += DEC_WARPS * 32) {
        const int h = u / HD, d = u - h * HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) m = fmaxf(m, s_ml[w][h][0]);
        float l = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) {
            const float f = s_ml[w][h][0] == -INFINITY ? (s_ml[w][h][1] == 0.f ? 0.f : 1.f) : exp2f(s_ml[w][h][0] - m);
            l += f * s_ml[w][h][1];
            x += f * so[(w * NH + h) * HD + d];
        }
        so[h * HD + d] = x;              // warp 0's place of this very number: nobody else reads it
        if (d == 0) { s_cta[h][0] = m; s_cta[h][1] = l; }
    }
    const unsigned C = cluster_size(), rank = cluster_rank();
    if (C > 1) cluster_sync(); else __syncthreads();
    const int range = blockIdx.x / C;
    for (int u = rank * DEC_WARPS * 32 + tid; u < nh * HD; u += C * DEC_WARPS * 32) {
        const int h = u / HD, d = u - h * HD;
        float m, l, x;
        if (C == 1) {
            m = s_cta[h][0]; l = s_cta[h][1]; x = so[u];
        } else {
            m = -INFINITY;
            for (unsigned c = 0; c < C; c++) m = fmaxf(m, peer_load(&s_cta[h][0], c));
            l = 0.f; x = 0.f;
            for (unsigned c = 0; c < C; c++) {
                const float mc = peer_load(&s_cta[h][0], c), lc = peer_load(&s_cta[h][1], c);
                const float f = mc == -INFINITY ? (lc == 0.f ? 0.f : 1.f) : exp2f(mc - m);
                l += f * lc;
                x += f * peer_load(so + u, c);
            }
        }
        const int64_t at = (int64_t)token * a.n_heads + head0 + h;
        if (a.ranges == 1) {
            reinterpret_cast<T*>(a.out)[at * HD + d] = from_f32<T>(l == 0.f ? 0.f : x / l);
        } else {
            a.part_o[(at * a.ranges + range) * HD + d] = x;
            if (d == 0) {
                a.part_ml[(at * a.ranges + range) * 2] = m;
                a.part_ml[(at * a.ranges + range) * 2 + 1] = l;
            }
        }
    }
    if (C > 1) cluster_sync();           // nobody leaves while another still reads its shared memory
}

// joins the ranges of a (token, head) in order
template <typename T>
__global__ void __launch_bounds__(HD) attn_decode_q8_join_kernel(T* __restrict__ out, const float* __restrict__ part_o,
                                                                 const float* __restrict__ part_ml, int ranges) {
    griddep_wait();
    griddep_launch();
    const int64_t at = blockIdx.x;
    const int d = threadIdx.x;
    float m = -INFINITY;
    for (int r = 0; r < ranges; r++) m = fmaxf(m, part_ml[(at * ranges + r) * 2]);
    float l = 0.f, x = 0.f;
    for (int r = 0; r < ranges; r++) {
        const float mr = part_ml[(at * ranges + r) * 2], lr = part_ml[(at * ranges + r) * 2 + 1];
        const float f = mr == -INFINITY ? (lr == 0.f ? 0.f : 1.f) : exp2f(mr - m);
        l += f * lr;
        x += f * part_o[(at * ranges + r) * HD + d];
    }
    out[at * HD + d] = from_f32<T>(l == 0.f ? 0.f : x / l);
}

template <typename T, int NG>
int launch_decode(const DecodeArgs& a, int n_tokens, int cluster, cudaStream_t stream) {
    constexpr size_t smem = (size_t)HD / 16 * Parts<T>::Q * NG * 32 * 8 + (size_t)DEC_WARPS * 8 * NG * HD * 4;
    static_assert(smem <= 227 * 1024, "shared memory");
    auto kernel = attn_decode_q8_kernel<T, NG>;
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.ranges * cluster, a.n_kv * a.subs, n_tokens);
        cfg.blockDim = dim3(DEC_WARPS * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = kllm_pdl_enabled() ? 2 : 1;
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(g_kllm_err, sizeof(g_kllm_err), "attention (8 bits): launch of the decode kernel: %s", cudaGetErrorString(e));
        return (int)e;
    }
    if (a.ranges > 1) {
        kllm_launch((attn_decode_q8_join_kernel<T>), dim3(n_tokens * a.n_heads), dim3(HD), 0, stream, (T*)a.out, (const float*)a.part_o,
                    (const float*)a.part_ml, a.ranges);
    }
    KLLM_LAUNCH_STATUS();
}

// ---- portions of prompts -------------------------------------------------------------------------------------------------
//
// A CTA takes 64 rows = (tokens of one request's portion) x (heads of one kv group), 16 a warp, and walks the portion's keys
// in tiles of 64.  A tile is converted to float16 once, on its way into shared memory, and read from there by all warps
// as operands (ldmatrix); the next tile's bytes are in registers meanwhile.  Weights go from the first product's result to
// the second's operand in registers.

constexpr int PRE_ROWS = 64, PRE_KEYS = 64, PRE_THREADS = 128;
constexpr int PRE_LD = HD + 8;                            // halves of a row in shared memory: eight rows on eight bank groups

__device__ __forceinline__ void ldmatrix4(unsigned addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(unsigned addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

struct PrefillArgs {
    void* out;
    const void* q;
    int64_t q_stride;
    const uint8_t* kcache;
    const uint8_t* vcache;
    const float* kscale;
    const float* vscale;
    const int* q_start;
    const int* start_pos;
    const int* block_table;
    int max_blocks, n_pages, n_tokens, n_requests, n_heads, n_kv, page_size, window, tokens_per_tile;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(PRE_THREADS) attn_prefill_q8_kernel(const PrefillArgs a) {
    constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
    constexpr int PIECES = HD / 16;                       // 16-byte pieces of a stored row
    constexpr int LOADS = PRE_KEYS * PIECES / PRE_THREADS;   // pieces of K (and of V) a thread carries
    static_assert(PRE_KEYS * PIECES % PRE_THREADS == 0, "pieces per thread");
    extern __shared__ __align__(16) unsigned char smem[];
    __half* sq = reinterpret_cast<__half*>(smem);                     // [NQ][rows][PRE_LD]
    __half* sk = sq + NQ * PRE_ROWS * PRE_LD;                         // [keys][PRE_LD]
    __half* sv = sk + PRE_KEYS * PRE_LD;
    __shared__ float s_mul[PRE_KEYS], s_ev[PRE_KEYS], s_inv[PRE_KEYS];   // per key: 2^ek, ev (-inf: not there), 2^-ev
    __shared__ int s_row[PRE_KEYS];
    __shared__ float s_factor[PRE_ROWS];
    __shared__ int s_req, s_tok0;
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x % a.n_kv, gs = a.n_heads / a.n_kv;
    if (tid == 0) {
        int tile = (gridDim.x - 1 - blockIdx.x) / a.n_kv, req = -1, tok0 = 0;       // longest key ranges first
        for (int s = 0; s < a.n_requests; s++) {
            const int n = a.q_start[s + 1] - a.q_start[s];
            const int nt = (n + a.tokens_per_tile - 1) / a.tokens_per_tile;
            if (tile < nt) { req = s; tok0 = a.q_start[s] + tile * a.tokens_per_tile; break; }
            tile -= nt;
        }
        s_req = req; s_tok0 = tok0;
    }
    __syncthreads();
    const int req = s_req, tok0 = s_tok0;
    if (req < 0) return;                                  // the grid is an upper bound on the tiles
    const int n_tok = min(min(a.tokens_per_tile, a.q_start[req + 1] - tok0), a.n_tokens - tok0);
    if (n_tok <= 0) return;
    const int pos0 = a.start_pos[req] + (tok0 - a.q_start[req]);
    const int lo = (a.window > 0 && pos0 + 1 > a.window) ? pos0 + 1 - a.window : 0;
    const int hi = pos0 + n_tok;
    const int* table = a.block_table + (int64_t)req * a.max_blocks;

    // queries into shared memory as float16 parts; a quarter warp's lanes share a row's pieces
    const T* q = (const T*)a.q;
    for (int r = warp * 16; r < warp * 16 + 16; r++) {
        const int tt = r / gs, hh = r - tt * gs;
        const bool ok = tt < n_tok && r < a.tokens_per_tile * gs;
        const T* src = q + (int64_t)(tok0 + tt) * a.q_stride + (int64_t)(kvh * gs + hh) * HD;
        float x[HD / 32];
        int m = 0;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            x[i] = ok ? to_f32(src[i * 32 + lane]) : 0.f;
            m = max(m, __float_as_int(x[i]) & 0x7fffffff);
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const bool finite = m < 0x7f800000;
        const float up = q8_pow2(row_shift(finite ? m : 0));
        if (lane == 0) s_factor[r] = finite ? a.scale * kLog2e * q8_pow2(-row_shift(m)) : __int_as_float(0x7fffffff);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            __half parts[NQ];
            split<NQ>(finite ? x[i] * up : 0.f, parts);
#pragma unroll
            for (int j = 0; j < NQ; j++) sq[(j * PRE_ROWS + r) * PRE_LD + i * 32 + lane] = parts[j];
        }
    }
    __syncwarp();
    int p_row[2];
    float factor[2], m_ref[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = warp * 16 + i * 8 + g8, tt = r / gs;
        p_row[i] = (tt < n_tok && r < a.tokens_per_tile * gs) ? pos0 + tt : -1;
        factor[i] = s_factor[r];
    }
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] = 0.f;

    const int first = lo / PRE_KEYS, last = (hi + PRE_KEYS - 1) / PRE_KEYS;
    uint4 kv[2][LOADS];
    int next_row = -1;
    float next_mul = 0.f, next_ev = -INFINITY, next_inv = 0.f;
    auto lookup = [&](int tile) {                         // threads 0..63: one key each
        next_row = -1; next_mul = 0.f; next_ev = -INFINITY; next_inv = 0.f;
        const int key = tile * PRE_KEYS + tid;
        if (tid >= PRE_KEYS || key < lo || key >= hi) return;
        const int lp = key / a.page_size;
        if (lp >= a.max_blocks) return;
        const int page = table[lp];
        if ((unsigned)page >= (unsigned)a.n_pages) return;
        const int cell = page * a.n_kv + kvh;
        next_row = cell * a.page_size + key - lp * a.page_size;
        next_mul = a.kscale[cell];
        const int e = q8_exponent(a.vscale[cell]);
        next_ev = (float)e;
        next_inv = q8_pow2(-e);
    };
    auto request = [&]() {                                // the tile whose rows are in s_row, into registers
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int u = tid + i * PRE_THREADS, key = u / PIECES, piece = u - key * PIECES;
            const int r = s_row[key];
            kv[0][i] = kv[1][i] = make_uint4(0, 0, 0, 0);
            if (r >= 0) {
                kv[0][i] = __ldg(reinterpret_cast<const uint4*>(a.kcache + (int64_t)r * HD + piece * 16));
                kv[1][i] = __ldg(reinterpret_cast<const uint4*>(a.vcache + (int64_t)r * HD + piece * 16));
            }
        }
    };
    lookup(first);
    if (tid < PRE_KEYS) s_row[tid] = next_row;
    __syncthreads();
    if (first < last) request();
    const unsigned sq_u = (unsigned)__cvta_generic_to_shared(sq), sk_u = (unsigned)__cvta_generic_to_shared(sk);
    const unsigned sv_u = (unsigned)__cvta_generic_to_shared(sv);
    // this lane's row address for ldmatrix: A tiles (16 x 16), and pairs of B tiles
    const unsigned a_off = (unsigned)(((warp * 16 + (lane & 15)) * PRE_LD + (lane >> 4) * 8) * 2);
    const unsigned kb_off = (unsigned)((((lane >> 4) * 8 + (lane & 7)) * PRE_LD + ((lane >> 3) & 1) * 8) * 2);
    const unsigned vb_off = (unsigned)((((lane & 15)) * PRE_LD + (lane >> 4) * 8) * 2);
    for (int tile = first; tile < last; tile++) {
        __syncthreads();                                  // the tile before has been used
        if (tid < PRE_KEYS) { s_mul[tid] = next_mul; s_ev[tid] = next_ev; s_inv[tid] = next_inv; }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int u = tid + i * PRE_THREADS, key = u / PIECES, piece = u - key * PIECES;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const uint4 x = kv[w][i];
                uint4 lo4, hi4;
                lo4.x = q8_to_f16x2(x.x & 0xffffu); lo4.y = q8_to_f16x2(x.x >> 16); lo4.z = q8_to_f16x2(x.y & 0xffffu); lo4.w = q8_to_f16x2(x.y >> 16);
                hi4.x = q8_to_f16x2(x.z & 0xffffu); hi4.y = q8_to_f16x2(x.z >> 16); hi4.z = q8_to_f16x2(x.w & 0xffffu); hi4.w = q8_to_f16x2(x.w >> 16);
                uint4* dst = reinterpret_cast<uint4*>((w ? sv : sk) + key * PRE_LD + piece * 16);
                dst[0] = lo4; dst[1] = hi4;
            }
        }
        lookup(tile + 1);
        if (tid < PRE_KEYS) s_row[tid] = next_row;
        __syncthreads();
        if (tile + 1 < last) request();
        float s[PRE_KEYS / 8][4];
#pragma unroll
        for (int i = 0; i < PRE_KEYS / 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
            uint32_t qa[NQ][4];
#pragma unroll
            for (int j = 0; j < NQ; j++) ldmatrix4(sq_u + (unsigned)(j * PRE_ROWS * PRE_LD * 2) + a_off + kk * 32, qa[j]);
#pragma unroll
            for (int n = 0; n < PRE_KEYS / 16; n++) {
                uint32_t b[4];
                ldmatrix4(sk_u + kb_off + (unsigned)(n * 16 * PRE_LD * 2) + kk * 32, b);
#pragma unroll
                for (int j = NQ - 1; j >= 0; j--) {
                    mma16816(s[2 * n], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b[0], b[1]);
                    mma16816(s[2 * n + 1], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b[2], b[3]);
                }
            }
        }
        const int key0 = tile * PRE_KEYS;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < PRE_KEYS / 8; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int kx = n * 8 + 2 * t4 + j, key = key0 + kx;
                const float mul = s_mul[kx], ev = s_ev[kx];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float& x = s[n][2 * i + j];
                    x = fmaf(x * mul, factor[i], ev);
                    if (key > p_row[i] || (a.window > 0 && key + a.window <= p_row[i]) || ev == -INFINITY) x = -INFINITY;
                    mx[i] = fmaxf(mx[i], x);
                }
            }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            if (mx[i] > m_ref[i] + kMoveAt) {
                const float corr = m_ref[i] == -INFINITY ? 0.f : exp2f(m_ref[i] - mx[i]);
                m_ref[i] = mx[i];
                l_run[i] *= corr;
#pragma unroll
                for (int n = 0; n < HD / 8; n++) { o[n][2 * i] *= corr; o[n][2 * i + 1] *= corr; }
            }
        }
        const float ref[2] = {m_ref[0] == -INFINITY ? 0.f : m_ref[0] - kLift, m_ref[1] == -INFINITY ? 0.f : m_ref[1] - kLift};
#pragma unroll
        for (int n = 0; n < PRE_KEYS / 8; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float inv = s_inv[n * 8 + 2 * t4 + j];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float& x = s[n][2 * i + j];
                    x = fast_exp2(x - ref[i]);
                    l_run[i] = fmaf(x, inv, l_run[i]);
                }
            }
#pragma unroll
        for (int kk = 0; kk < PRE_KEYS / 16; kk++) {
            uint32_t pa[NP][4];
#pragma unroll
            for (int x = 0; x < 4; x++) {                 // a0: row g, keys 2t; a1: row g + 8; a2, a3: keys + 8
                const int n = 2 * kk + (x >> 1), i = x & 1;
                __half h0[NP], h1[NP];
                split<NP>(s[n][2 * i], h0);
                split<NP>(s[n][2 * i + 1], h1);
#pragma unroll
                for (int j = 0; j < NP; j++) {
                    const __half2 hh = __halves2half2(h0[j], h1[j]);
                    pa[j][x] = *reinterpret_cast<const uint32_t*>(&hh);
                }
            }
#pragma unroll
            for (int n = 0; n < HD / 16; n++) {
                uint32_t b[4];
                ldmatrix4t(sv_u + vb_off + (unsigned)(kk * 16 * PRE_LD * 2) + n * 32, b);
#pragma unroll
                for (int j = NP - 1; j >= 0; j--) {
                    mma16816(o[2 * n], pa[j][0], pa[j][1], pa[j][2], pa[j][3], b[0], b[1]);
                    mma16816(o[2 * n + 1], pa[j][0], pa[j][1], pa[j][2], pa[j][3], b[2], b[3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
        const int r = warp * 16 + i * 8 + g8, tt = r / gs, hh = r - tt * gs;
        if (tt >= n_tok || r >= a.tokens_per_tile * gs) continue;
        T* dst = (T*)a.out + ((int64_t)(tok0 + tt) * a.n_heads + kvh * gs + hh) * HD;
#pragma unroll
        for (int n = 0; n < HD / 8; n++) {
            const float x = l_run[i] == 0.f ? 0.f : o[n][2 * i] / l_run[i], y = l_run[i] == 0.f ? 0.f : o[n][2 * i + 1] / l_run[i];
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<__nv_bfloat162*>(dst + n * 8 + 2 * t4) = __floats2bfloat162_rn(x, y);
            } else {
                *reinterpret_cast<float2*>(dst + n * 8 + 2 * t4) = make_float2(x, y);
            }
        }
    }
}

template <typename T> int launch_prefill(const PrefillArgs& a, cudaStream_t stream) {
    constexpr size_t smem = (size_t)(Parts<T>::Q * PRE_ROWS + 2 * PRE_KEYS) * PRE_LD * 2;
    static_assert(smem <= 226 * 1024, "shared memory");
    const cudaError_t e = cudaFuncSetAttribute(attn_prefill_q8_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(g_kllm_err, sizeof(g_kllm_err), "attention (8 bits): %zu bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
        return (int)e;
    }
    const int tiles = a.n_tokens / a.tokens_per_tile + a.n_requests;
    kllm_launch((attn_prefill_q8_kernel<T>), dim3((unsigned)tiles * a.n_kv), dim3(PRE_THREADS), smem, stream, a);
    KLLM_LAUNCH_STATUS();
}

int check_common(int n_heads, int n_kv, int hd, int page_size, int n_pages, int dtype, const void* out, const void* kcache,
                 const void* vcache) {
    if (hd != HD) KLLM_FAIL("attention (8 bits): this library was built for head size %d, not %d", HD, hd);
    if (n_kv <= 0 || n_heads <= 0 || n_heads % n_kv) KLLM_FAIL("attention (8 bits): %d heads over %d kv heads", n_heads, n_kv);
    if (page_size <= 0) KLLM_FAIL("attention (8 bits): page size %d", page_size);
    if (n_pages <= 0) KLLM_FAIL("attention (8 bits): a cache of %d pages", n_pages);
    if ((int64_t)n_pages * n_kv * page_size >= (1LL << 31)) KLLM_FAIL("attention (8 bits): a store of 2^31 rows or more");
    if (dtype != KLLM_F32 && dtype != KLLM_BF16) KLLM_FAIL("attention (8 bits): element type %d", dtype);
    if ((((uintptr_t)kcache | (uintptr_t)vcache) & 15) || ((uintptr_t)out & 7))
        KLLM_FAIL("attention (8 bits): the caches must be 16-byte aligned, out 8-byte");
    return 0;
}

}  // namespace

extern "C" int kllm_attention_q8_head_dim() { return HD; }

// One row per token: token t of request token_req[t] (NULL: request t) at positions[t] sees its request's keys up to its
// own place.  out [n, heads*HD] in dtype; parts: float32 [n, heads, ranges, HD] and [n, heads, ranges, 2] where ranges > 1.
// A context is cut into ranges * cluster parts.
extern "C" int kllm_attention_decode_q8(void* out, float* part_o, float* part_ml, const void* q, int64_t q_stride,
                                        const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                                        const int* positions, const int* token_req, const int* block_table, int max_blocks,
                                        int n_pages, int n_tokens, int n_requests, int n_heads, int n_kv, int hd, int page_size,
                                        int window, float scale, int ranges, int cluster, int dtype, void* stream) {
    if (n_tokens <= 0) return 0;
    const int rc = check_common(n_heads, n_kv, hd, page_size, n_pages, dtype, out, kcache, vcache);
    if (rc) return rc;
    if (ranges < 1 || (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8))
        KLLM_FAIL("attention (8 bits): %d ranges of clusters of %d CTAs", ranges, cluster);
    if (ranges > 1 && (!part_o || !part_ml)) KLLM_FAIL("attention (8 bits): several ranges without room for their parts");
    if (n_tokens > 65535) KLLM_FAIL("attention (8 bits): %d tokens in one launch, at most 65535", n_tokens);
    // the heads of a group in equal parts of at most 16 (8 where the accumulators of 16 do not fit the registers)
    const int gs = n_heads / n_kv, most = HD <= 128 ? 16 : 8;
    int subs = 1;
    while (gs % subs || gs / subs > most) subs++;
    if ((int64_t)n_kv * subs > 65535) KLLM_FAIL("attention (8 bits): %d kv heads in %d parts each", n_kv, subs);
    DecodeArgs a{out, part_o, part_ml, q, q_stride, (const uint8_t*)kcache, (const uint8_t*)vcache, kscale, vscale, positions,
                 token_req, block_table, max_blocks, n_pages, n_requests, n_heads, n_kv, subs, gs / subs, page_size,
                 window > 0 ? window : 0, ranges, scale};
    const cudaStream_t s = (cudaStream_t)stream;
    if constexpr (HD <= 128) {
        if (a.heads_per_cta > 8)
            return dtype == KLLM_F32 ? launch_decode<float, 2>(a, n_tokens, cluster, s) : launch_decode<bf16, 2>(a, n_tokens, cluster, s);
    }
    return dtype == KLLM_F32 ? launch_decode<float, 1>(a, n_tokens, cluster, s) : launch_decode<bf16, 1>(a, n_tokens, cluster, s);
}

// Requests' portions: rows q_start[s]..q_start[s+1] of request s start at cache position start_pos[s].
extern "C" int kllm_attention_prefill_q8(void* out, const void* q, int64_t q_stride, const void* kcache, const void* vcache,
                                         const float* kscale, const float* vscale, const int* q_start, const int* start_pos,
                                         const int* block_table, int max_blocks, int n_pages, int n_tokens, int n_requests,
                                         int n_heads, int n_kv, int hd, int page_size, int window, float scale, int dtype,
                                         void* stream) {
    if (n_tokens <= 0 || n_requests <= 0) return 0;
    const int rc = check_common(n_heads, n_kv, hd, page_size, n_pages, dtype, out, kcache, vcache);
    if (rc) return rc;
    const int gs = n_heads / n_kv;
    if (gs > PRE_ROWS) KLLM_FAIL("attention (8 bits): %d heads per kv head, at most %d", gs, PRE_ROWS);
    PrefillArgs a{out, q, q_stride, (const uint8_t*)kcache, (const uint8_t*)vcache, kscale, vscale, q_start, start_pos, block_table,
                  max_blocks, n_pages, n_tokens, n_requests, n_heads, n_kv, page_size, window > 0 ? window : 0, PRE_ROWS / gs, scale};
    return dtype == KLLM_F32 ? launch_prefill<float>(a, (cudaStream_t)stream) : launch_prefill<bf16>(a, (cudaStream_t)stream);
}
