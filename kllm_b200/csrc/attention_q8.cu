// Causal grouped-query attention over the paged cache in 8 bits (q8.cuh), one library per head size (-DKLLM_HD, a multiple
// of 32 up to 256).  Queries and outputs are bfloat16 or float32.
//
// For a row (the token at position p, head h over kv head g) and the keys j it sees, max(0, p + 1 - window) <= j <= p:
//     s_j = log2(e) scale (q . k8_j) 2^ek(j),      weight 2^s_j / sum,      out = sum_j weight_j v8_j 2^ev(j)
// where ek, ev are the exponents of the page's scales.  A value page's exponent goes into the weight's: with a reference M,
//     w_j = 2^(s_j + ev(j) - M + 7),   l = sum_j w_j 2^-ev(j),   O = sum_j w_j v8_j,   out = O / l,
// so that one exponential a score serves both sums, whatever the pages' scales are.  The reference follows the running
// maximum of s_j + ev(j) and is moved only when that has grown by more than 7.875: w stays below 2^15, a float16 number, and
// what is smaller than 2^-32 of the largest weight is lost.
//
// Products run on the tensor cores in float16 with float32 sums (mma.sync m16n8k16): e4m3 numbers are float16 numbers.
// A row of bfloat16 queries is one float16 operand, exactly, after division by a power of two that brings its largest
// magnitude to 2^14..2^15; a float32 row is the sum of three (33 bits).  Weights are one float16 (11 bits: half a step is
// 2^-12, against bfloat16's 2^-9), beside float32 queries two (22 bits).  A row with an infinity or NaN among its queries
// becomes NaN, if it sees a key.
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
template <typename T> struct Parts { static constexpr int Q = 1, P = 1; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 2; };

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ... of a sum that begins
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// part i of x: x = p0 + p1 + p2 + ..., each a float16 number
template <int N> __device__ __forceinline__ void split(float x, __half (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        p[i] = __float2half_rn(x);
        x -= __half2float(p[i]);
    }
}

// part i, 0 behind the last
template <int N> __device__ __forceinline__ __half pick(const __half (&p)[N], int i) {
    __half x = __ushort_as_half(0);
#pragma unroll
    for (int j = 0; j < N; j++)
        if (i == j) x = p[j];
    return x;
}

// ---- single tokens ---------------------------------------------------------------------------------------------------
//
// What bounds it: bytes.  Every warp walks its own tiles of keys, which it requests ahead into a ring of its own in shared
// memory (cp.async), without meeting other warps.  The tensor core's operands are read from there as they lie: keys are
// the M side (A, 16 keys x 16 dims), the heads of the group the N side (8 at a time); lane (g, t) = (lane / 4, lane % 4)
// holds rows g and g + 8, and because the order of the dims under a sum is free, its dims are 16 neighbours of every 64
// (one 16-byte read), the same for the queries.  The second product takes values as A with the dims as M: lane (g, t)
// holds HD / 8 neighbouring dims of rows 2t, 2t + 1, 2t + 8, 2t + 9; two rows' bytes are interleaved (prmt) and converted
// to the pairs that the operand wants, and the weights, whose layout is (key, head), become the B operand by an 8 x 8
// transposition in registers (movmatrix).  Row r of a tile is key r ^ (r >> 1 & 1) of it, and the 16-byte pieces of key j lie
// at piece ^ swizzle(j): with both, neither kind of read meets a bank twice at head sizes 64 and 128.
//
// Measured, back to back, bfloat16 (% of a copy's 6.45 TB/s): 64 requests of 846 to 4095 keys, 32 heads over 8 of 128, pages of 16: 69.9 us (72 %);
// one of 131072 keys 54.2 us (77 %); 8 of 2048 keys, 32 over 4 of 64: 8.6 us; one: 6.2 us, a chain of launch, table, tiles and
// joins.  Float32, 5 requests of 604 to 1501 keys, 32 heads of 128: 17.8 us (37 %).  With loads straight into registers the
// first took 131 us: a warp then waits for each of its tiles.  Eight warps a CTA at head size 64 (16 of a CTA pair an SM as before): 64 x 2048
// keys 18.7 us against 19.6, 128 x 1000 23.0 against 18.8.

constexpr int DEC_KT = HD <= 128 ? 32 : 16;              // keys of a warp's tile
constexpr int DEC_MT = DEC_KT / 16;
constexpr int DEC_WARPS = 4;
constexpr int DEC_STAGES = HD <= 32 ? 4 : HD <= 64 ? 3 : 2;
constexpr int KW = HD % 64 == 0 ? 4 : 2;                 // words of a lane's piece of a key row
constexpr int KC = HD / (16 * KW);                       // pieces of a key row (16 * KW dims each)
constexpr int VW = HD / 32;                              // words of a lane's piece of a value row
constexpr int PIECES = HD / 16;                          // 16-byte pieces of a row
constexpr int DEC_TILE = DEC_KT * HD;                    // bytes of a tile of keys (or values)
constexpr int DEC_META = DEC_KT * 8;                     // a tile's scales: (key scale, value scale) per key, then what is made of them
constexpr int DEC_RING = DEC_STAGES * 2 * DEC_TILE + (DEC_STAGES + 1) * DEC_META;

__device__ __forceinline__ int dec_swizzle(int key) {
    return PIECES == 8 || PIECES == 16 ? (key & 6) ^ ((key & 1) << 2) : PIECES == 4 ? (key >> 1) & 2 : 0;
}
__device__ __forceinline__ int dec_key(int row) { return row ^ ((row >> 1) & 1); }

// SPREAD: where a CTA has one or two heads of float32 queries, the parts of a head's queries, and of its weights, are columns
// of the N side (part p of head h is column 2 p + h) instead of products of their own: a third of the first product's
// instructions and half of the second's (32 heads of 128, 8 x 2048 keys: 36.7 us against more than 40).  Three or four heads: the
// weights' parts alone (part p of head h is column 4 p + h; both columns have the head's queries): 64 x 2048 keys of 32 heads over 8
// of 128 60.8 us, with two products 85, of which most is what registers were missing.
template <typename T, int NG, int SPREAD> struct DecodeShape {
    static constexpr int NQ = SPREAD == 2 ? 1 : Parts<T>::Q;
    static constexpr int QREGS = HD / 16 * 2 * NQ * NG;
    static constexpr bool Q_IN_REGS = QREGS <= 32;
    static constexpr int Q_BYTES = Q_IN_REGS ? 0 : HD / 16 * NQ * NG * 32 * 8;
    static constexpr int SUM_BYTES = DEC_WARPS * 8 * NG * HD * 4;     // over the rings, when they are done with
    static constexpr int SMEM = Q_BYTES + (DEC_WARPS * DEC_RING > SUM_BYTES ? DEC_WARPS * DEC_RING : SUM_BYTES);
    // CTAs an SM, by shared memory and registers
    static constexpr int CTAS = HD <= 64 ? 4 : HD <= 128 ? 3 : 2;
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
    bool q_by_four;              // rows of queries may be read four numbers at a time
    float scale;
};

// four numbers of a row of queries, zeros where the row is none
template <typename T> __device__ __forceinline__ void load4(const T* p, bool there, bool by_four, float (&x)[4]) {
    x[0] = x[1] = x[2] = x[3] = 0.f;
    if (!there) return;
    if (!by_four) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_f32(p[i]);
    } else if constexpr (sizeof(T) == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float4 w = *reinterpret_cast<const float4*>(p);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    }
}
template <int W> __device__ __forceinline__ void read_words(unsigned addr, uint32_t* r) {
    if constexpr (W == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
    else if constexpr (W == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
    else asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(r[0]) : "r"(addr));
}
// bytes 16, or 0: the place is filled with zeros
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

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
// ... in two: what this thread did before the arrival is done when the others are past their wait
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory"); }
__device__ __forceinline__ unsigned peer_addr(const void* p, unsigned rank) {
    unsigned b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(b) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    return b;
}
__device__ __forceinline__ float2 peer_load2(const void* p, unsigned rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(peer_addr(p, rank)));
    return v;
}
__device__ __forceinline__ float4 peer_load4(const void* p, unsigned rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_addr(p, rank)));
    return v;
}
// grid: (ranges * cluster, kv heads * subgroups of heads, tokens), clusters along x; a cluster's CTAs take neighbouring
// parts of a range and join through distributed shared memory
template <typename T, int NG, int SPREAD>         // heads in their parts' columns: 2, 4, or 0: every part a product
__global__ void __launch_bounds__(DEC_WARPS * 32, (DecodeShape<T, NG, SPREAD>::CTAS))
attn_decode_q8_kernel(const DecodeArgs a) {
    using Shape = DecodeShape<T, NG, SPREAD>;
    constexpr int NQ = Shape::NQ, NP = SPREAD ? 1 : Parts<T>::P, NH = 8 * NG;
    constexpr bool Q_IN_REGS = Shape::Q_IN_REGS, WIDE = Parts<T>::Q > 1;
    static_assert(SPREAD == 0 || (WIDE && NG == 1 && (SPREAD == 2 ? Parts<T>::Q <= 4 && Parts<T>::P <= 4 : SPREAD == 4 && Parts<T>::P <= 2)),
                  "the parts of two or four heads are eight columns");
    extern __shared__ __align__(128) unsigned char smem[];
    uint2* sq = reinterpret_cast<uint2*>(smem);                       // the queries as operands: [kk][part][ng][lane]
    float* so = reinterpret_cast<float*>(smem + Shape::Q_BYTES);      // [warps][NH][HD], then the CTA's sum [NH][HD]
    __shared__ float s_ml[DEC_WARPS][NH][2];                          // references and sums of the warps
    __shared__ __align__(8) float s_cta[NH][2];                                    // ... of the CTA
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int token = blockIdx.z, kvh = blockIdx.y / a.subs, sub = blockIdx.y % a.subs;
    const int head0 = kvh * (a.n_heads / a.n_kv) + sub * a.heads_per_cta, nh = a.heads_per_cta;
    const int req = a.token_req ? a.token_req[token] : token;
    const int p = (req >= 0 && req < a.n_requests) ? a.positions[token] : -1;
    const int lo = (a.window > 0 && p >= a.window) ? p - a.window + 1 : 0, hi = keys_end((int64_t)p + 1, a.max_blocks, a.page_size);

    // this warp's tiles: the token's tiles [first, last) in one part per CTA, a part's tiles in turn over the warps
    const int parts = gridDim.x, part = blockIdx.x;
    const int first = lo / DEC_KT, last = (hi + DEC_KT - 1) / DEC_KT;      // tiles start at multiples of their size
    const int per = (max(last - first, 0) + parts - 1) / parts;
    const int tile_lo = first + part * per, tile_hi = min(last, tile_lo + per);

    const int* table = a.block_table + (int64_t)(req < 0 ? 0 : req) * a.max_blocks;
    // A lane looks after key tile * DEC_KT + lane % DEC_KT: its page (-1: not seen), read from the table a tile ahead of the
    // copies that need it, then its row in the stores.
    auto find = [&](int tile, int& page, int& slot) {
        page = -1; slot = 0;
        const int key = tile * DEC_KT + (lane & (DEC_KT - 1));
        if (tile >= tile_hi || key < lo || key >= hi) return;
        const int lp = key / a.page_size;
        slot = key - lp * a.page_size;
        if (lp < a.max_blocks) page = load_early(table + lp);
    };
    const unsigned ring = (unsigned)__cvta_generic_to_shared(smem) + Shape::Q_BYTES + warp * DEC_RING;
    const unsigned meta = ring + DEC_STAGES * 2 * DEC_TILE;
    // Copies of 16 bytes, COPIES a lane and tile.  Sixteen keys of one page, all seen, lie one behind the other: their
    // copies differ by constants, where a look-up per row costs a shuffle, a comparison and a 64-bit product each.
    constexpr int COPIES = DEC_KT * PIECES / 32;
    const bool blocks = a.page_size % 16 == 0;
    // Rows of the tile that is being requested, -1: not seen: of the lane's key, and of the keys whose pieces the lane copies (in blocks: the
    // first two are a row each).  The latter are handed over once where there are registers, else again for the values: a spilled register
    // is fetched from L2, as the rings leave no first-level cache.
    constexpr bool KEEP_ROWS = !WIDE && NG == 1;
    int row = -1, rows[KEEP_ROWS ? COPIES : 1];
    unsigned held = 0;                    // bit i: the lane's key of the i'th tile on its way is seen
    bool whole = false;
    auto request_rows = [&](unsigned dst, const uint8_t* store, auto is_key) {
        constexpr bool LOOK = decltype(is_key)::value || !KEEP_ROWS;
        if (whole) {
            const uint8_t* src[DEC_MT];
#pragma unroll
            for (int b = 0; b < DEC_MT; b++) {
                const int r = LOOK ? __shfl_sync(0xffffffffu, row, b * 16) : rows[KEEP_ROWS ? b : 0];
                if constexpr (KEEP_ROWS) rows[b] = r;
                src[b] = store + (int64_t)r * HD;
            }
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int u = i * 32 + lane, key = u / PIECES, piece = u % PIECES;
                const int b = DEC_MT == 2 ? (COPIES % 2 == 0 ? i / (COPIES / 2) : key >> 4) : 0;
                copy16(dst + key * HD + ((piece ^ dec_swizzle(key)) << 4), (b ? src[DEC_MT - 1] : src[0]) + (u * 16 - b * 16 * HD), true);
            }
        } else {
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int u = i * 32 + lane, key = u / PIECES, piece = u % PIECES;
                const int r = LOOK ? __shfl_sync(0xffffffffu, row, key) : rows[KEEP_ROWS ? i : 0];
                if constexpr (KEEP_ROWS) rows[i] = r;
                copy16(dst + key * HD + ((piece ^ dec_swizzle(key)) << 4), store + (int64_t)max(r, 0) * HD + piece * 16, r >= 0);
            }
        }
        copies_commit();
    };
    auto request_k = [&](int stage, int meta_slot, int page, int slot) {
        const bool there = (unsigned)page < (unsigned)a.n_pages;
        const int cell = there ? page * a.n_kv + kvh : 0;
        row = there ? cell * a.page_size + slot : -1;
        if (lane < DEC_KT) {
            copy4(meta + meta_slot * DEC_META + lane * 8, a.kscale + cell, there);
            copy4(meta + meta_slot * DEC_META + lane * 8 + 4, a.vscale + cell, there);
        }
        held |= (unsigned)there << (DEC_STAGES - 1);
        whole = blocks && __all_sync(0xffffffffu, there);
        request_rows(ring + stage * 2 * DEC_TILE, a.kcache, std::true_type{});
    };
    auto request_v = [&](int stage) { request_rows(ring + stage * 2 * DEC_TILE + DEC_TILE, a.vcache, std::false_type{}); };
    float o[HD / 16][NG][4];
#pragma unroll
    for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int ng = 0; ng < NG; ng++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][ng][j] = 0.f;

    int page[DEC_STAGES + 1], slot[DEC_STAGES + 1];
#pragma unroll
    for (int i = 0; i <= DEC_STAGES; i++) find(tile_lo + warp + i * DEC_WARPS, page[i], slot[i]);
#pragma unroll
    for (int i = 0; i < DEC_STAGES; i++) {
        held >>= 1;
        request_k(i, i, page[i], slot[i]);
        request_v(i);
    }
    // Queries, while the first tiles are on their way: lane (g, t) holds its dims of head g, four lanes a head.  What does not
    // fit the registers (the parts of float32 queries) goes through shared memory, a quarter by each warp.
    const T* q = (const T*)a.q + (int64_t)token * a.q_stride + (int64_t)head0 * HD;
    uint2 qr[Q_IN_REGS ? HD / 16 * NQ * NG : 1];
    float factor[NG][2], m_ref[NG][2], l_run[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ng++) {
        const int h = SPREAD ? g8 & (SPREAD - 1) : ng * 8 + g8;
        float x[HD / 16][4];
        int m = 0;
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
            // dims of the step's k = 2t, 2t + 1 and 2t + 8, 2t + 9: four neighbours of lane t's piece
            load4(q + h * HD + (kk / KW) * (16 * KW) + t4 * (4 * KW) + (kk % KW) * 4, h < nh, a.q_by_four, x[kk]);
#pragma unroll
            for (int i = 0; i < 4; i++) m = max(m, __float_as_int(x[kk][i]) & 0x7fffffff);
        }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const bool finite = m < 0x7f800000;
        const float up = finite ? q8_pow2(row_shift(m)) : 0.f;
        const float f = finite ? a.scale * kLog2e * q8_pow2(-row_shift(m)) : __int_as_float(0x7fffffff);   // NaN: the row is
#pragma unroll
        for (int i = 0; i < 2; i++) {
            factor[ng][i] = __shfl_sync(0xffffffffu, f, (SPREAD == 2 ? i : 2 * t4 + i) * 4);
            m_ref[ng][i] = -INFINITY;
            l_run[ng][i] = 0.f;
        }
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
            __half parts[4][NQ];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (SPREAD == 2) {
                    __half all[Parts<T>::Q];
                    split<Parts<T>::Q>(finite ? x[kk][i] * up : 0.f, all);
                    parts[i][0] = pick(all, g8 >> 1);
                } else {
                    split<NQ>(finite ? x[kk][i] * up : 0.f, parts[i]);
                }
            }
#pragma unroll
            for (int j = 0; j < NQ; j++) {
                const __half2 w0 = __halves2half2(parts[0][j], parts[1][j]), w1 = __halves2half2(parts[2][j], parts[3][j]);
                const uint2 w = make_uint2(*reinterpret_cast<const uint32_t*>(&w0), *reinterpret_cast<const uint32_t*>(&w1));
                const int at = (kk * NQ + j) * NG + ng;
                if constexpr (Q_IN_REGS) qr[at] = w;
                else if (kk % DEC_WARPS == warp) sq[at * 32 + lane] = w;
            }
        }
    }
    if constexpr (!Q_IN_REGS) __syncthreads();
    int page_next = page[DEC_STAGES], slot_next = slot[DEC_STAGES];   // of the tile that is requested next
    int stage = 0, meta_slot = 0;
    for (int tile = tile_lo + warp; tile < tile_hi; tile += DEC_WARPS) {
        const int page_now = page_next, slot_now = slot_next;
        find(tile + (DEC_STAGES + 1) * DEC_WARPS, page_next, slot_next);
        copies_wait<2 * DEC_STAGES - 1>();                            // this tile's keys and scales
        __syncwarp();
        const unsigned k_at = ring + stage * 2 * DEC_TILE, v_at = k_at + DEC_TILE;
        // The scales of the lane's key, in their place, as all lanes want them: 2^ek and 2^-ev by their exponents in one word, ev (-inf: not
        // seen).  What the scores need of them per key and lane is four instructions then.
        if (lane < DEC_KT) {
            float scales[2];
            const unsigned at = meta + meta_slot * DEC_META + lane * 8;
            read_words<2>(at, reinterpret_cast<uint32_t*>(scales));
            const int ev = q8_exponent(scales[1]);
            asm volatile("st.shared.v2.b32 [%0], {%1,%2};\n" ::"r"(at), "r"((q8_exponent(scales[0]) + 127) << 23 | (127 - ev) << 15),
                         "r"(__float_as_int((held & 1u) ? (float)ev : -INFINITY)) : "memory");
        }
        held >>= 1;
        float s[DEC_MT][NG][4], part[DEC_MT][NG][4];
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[mt][ng][j] = 0.f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint32_t kr[DEC_MT][2][KW];
#pragma unroll
            for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int key = mt * 16 + i * 8 + dec_key(g8);
                    const int piece = KW == 4 ? c * 4 + t4 : c * 2 + (t4 >> 1);
                    read_words<KW>(k_at + key * HD + ((piece ^ dec_swizzle(key)) << 4) + (KW == 4 ? 0 : (t4 & 1) * 8), kr[mt][i]);
                }
#pragma unroll
            for (int w = 0; w < KW; w++) {
                const int kk = c * KW + w;
                uint32_t ka[DEC_MT][4];
#pragma unroll
                for (int mt = 0; mt < DEC_MT; mt++) {
                    q8_to_f16x4(kr[mt][0][w], ka[mt][0], ka[mt][2]);
                    q8_to_f16x4(kr[mt][1][w], ka[mt][1], ka[mt][3]);
                }
                // The tensor core cuts its sums; beside float32 queries 32 products at a time are added to a sum in registers
                // (one sum over 256 dims was 2.7 times as far from 64 bits as float32 arithmetic).
                float (&to)[DEC_MT][NG][4] = WIDE ? part : s;
                if (WIDE && kk % 2 == 0) {
#pragma unroll
                    for (int i = 0; i < DEC_MT * NG * 4; i++) (&part[0][0][0])[i] = 0.f;
                }
#pragma unroll
                for (int j = NQ - 1; j >= 0; j--)                   // the smallest part first
#pragma unroll
                    for (int ng = 0; ng < NG; ng++) {
                        const int at = (kk * NQ + j) * NG + ng;
                        const uint2 b = Q_IN_REGS ? qr[Q_IN_REGS ? at : 0] : sq[at * 32 + lane];
#pragma unroll
                        for (int mt = 0; mt < DEC_MT; mt++) mma16816(to[mt][ng], ka[mt][0], ka[mt][1], ka[mt][2], ka[mt][3], b.x, b.y);
                    }
                if (WIDE && kk % 2 == 1) {
#pragma unroll
                    for (int i = 0; i < DEC_MT * NG * 4; i++) (&s[0][0][0])[i] += (&part[0][0][0])[i];
                }
            }
        }
        __syncwarp();                                                 // everybody has read this tile's keys
        request_k(stage, meta_slot == 0 ? DEC_STAGES : meta_slot - 1, page_now, slot_now);
        if constexpr (SPREAD == 2) {                  // the parts of a score: every lane of a row has both heads' then
#pragma unroll
            for (int i = 0; i < DEC_MT * 4; i++) {
                float& x = (&s[0][0][0])[i];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
            }
        }
        // scores, in units of log2, with the values' exponents
        bool grown = false;
        float inv[DEC_MT][2];                       // 2^-ev of the lane's keys
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint32_t made[2];
                read_words<2>(meta + meta_slot * DEC_META + (mt * 16 + i * 8 + dec_key(g8)) * 8, made);
                const float mul = __uint_as_float(made[0] & 0x7f800000u), ev = __uint_as_float(made[1]);
                inv[mt][i] = __uint_as_float(made[0] << 8 & 0x7f800000u);
#pragma unroll
                for (int ng = 0; ng < NG; ng++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float& x = s[mt][ng][2 * i + j];
                        x = ev != -INFINITY ? fmaf(x * mul, factor[ng][j], ev) : -INFINITY;
                        grown = grown || x > moves_above(m_ref[ng][j]);
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
                    if (mx > moves_above(m_ref[ng][j])) {              // the same for every lane of the head
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
                    if constexpr (SPREAD) {
                        __half all[2][Parts<T>::P];
                        split<Parts<T>::P>(w[0], all[0]);
                        split<Parts<T>::P>(w[1], all[1]);
                        h0[0] = pick(all[0], SPREAD == 2 ? t4 : t4 >> 1);
                        h1[0] = pick(all[1], SPREAD == 2 ? t4 : t4 >> 1);
                    } else {
                        split<NP>(w[0], h0);
                        split<NP>(w[1], h1);
                    }
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        const __half2 hh = __halves2half2(h0[k], h1[k]);
                        pb[mt][k][ng][i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hh));
                    }
                }
        copies_wait<2 * DEC_STAGES - 1>();                            // this tile's values
        __syncwarp();
#pragma unroll
        for (int mt = 0; mt < DEC_MT; mt++) {
            uint32_t vr[4][VW];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = mt * 16 + (i >> 1) * 8 + dec_key(2 * t4 + (i & 1)), f = dec_swizzle(key);
                const unsigned at = v_at + key * HD;
                if constexpr (HD == 64) {
                    read_words<2>(at + (((g8 >> 1) ^ f) << 4) + (g8 & 1) * 8, vr[i]);
                } else if constexpr (HD % 128 == 0) {
#pragma unroll
                    for (int w = 0; w < VW; w += 4) read_words<4>(at + ((g8 * (VW / 4) + w / 4) ^ f) * 16, vr[i] + w);
                } else {
#pragma unroll
                    for (int w = 0; w < VW; w++) read_words<1>(at + g8 * (HD / 8) + w * 4, vr[i] + w);
                }
            }
#pragma unroll
            for (int w = 0; w < VW; w++) {
                uint32_t va[2][4];                                  // dims 4w, 4w + 1, then 4w + 2, 4w + 3
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const unsigned sel = half ? 0x7362u : 0x5140u;
                    const uint32_t x = __byte_perm(vr[0][w], vr[1][w], sel), y = __byte_perm(vr[2][w], vr[3][w], sel);
                    q8_to_f16x4(x, va[half][0], va[half][1]);
                    q8_to_f16x4(y, va[half][2], va[half][3]);
                }
                if constexpr (!WIDE) {
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int ng = 0; ng < NG; ng++)
                            mma16816(o[2 * w + half][ng], va[half][0], va[half][1], va[half][2], va[half][3], pb[mt][0][ng][0], pb[mt][0][ng][1]);
                } else {
                    // Beside float32 queries sixteen keys at a time are added to a sum in registers: what the tensor core cuts off one long
                    // sum added up, over 16001 keys, to three to five times float32 arithmetic's error.  It costs 2 to 8 %, with seven
                    // or eight heads of 128 a CTA 10 to 18.
                    float sum[2][NG][4];
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--)
#pragma unroll
                        for (int half = 0; half < 2; half++)
#pragma unroll
                            for (int ng = 0; ng < NG; ng++) {
                                if (k == NP - 1) mma16816_first(sum[half][ng], va[half][0], va[half][1], va[half][2], va[half][3], pb[mt][k][ng][0], pb[mt][k][ng][1]);
                                else mma16816(sum[half][ng], va[half][0], va[half][1], va[half][2], va[half][3], pb[mt][k][ng][0], pb[mt][k][ng][1]);
                            }
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int ng = 0; ng < NG; ng++)
#pragma unroll
                            for (int j = 0; j < 4; j++) o[2 * w + half][ng][j] += sum[half][ng][j];
                }
            }
        }
        __syncwarp();                                                 // everybody has read this tile's values
        request_v(stage);
        stage = stage + 1 == DEC_STAGES ? 0 : stage + 1;
        meta_slot = meta_slot == DEC_STAGES ? 0 : meta_slot + 1;
    }
    copies_wait<0>();
    __syncthreads();                                                  // the rings become the room for the sums

    // join: the warps of the CTA in order, then the CTAs of the cluster in order
#pragma unroll
    for (int ng = 0; ng < NG; ng++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l_run[ng][j] += __shfl_xor_sync(0xffffffffu, l_run[ng][j], d);
            const int h = SPREAD == 2 ? j : ng * 8 + 2 * t4 + j;
            const bool mine = SPREAD == 0 || 2 * t4 < SPREAD;         // of the lanes that hold the head's columns, the first
            if (g8 == 0 && mine) { s_ml[warp][h][0] = m_ref[ng][j]; s_ml[warp][h][1] = l_run[ng][j]; }
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
                // dims of rows g and g + 8 of step i: neighbours g * HD / 8 + 2 i, + 1
                float2 v = make_float2(o[i][ng][j], o[i][ng][2 + j]);
                if constexpr (SPREAD) {
                    v.x += __shfl_xor_sync(0xffffffffu, v.x, SPREAD / 2);
                    v.y += __shfl_xor_sync(0xffffffffu, v.y, SPREAD / 2);
                }
                if (mine) *reinterpret_cast<float2*>(so + ((warp * NH + h) * HD + g8 * (HD / 8) + 2 * i)) = v;
            }
        }
    __syncthreads();
    for (int u = tid; u < nh * (HD / 4); u += DEC_WARPS * 32) {
        const int h = u / (HD / 4), d = (u - h * (HD / 4)) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) m = fmaxf(m, s_ml[w][h][0]);
        float l = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) {
            const float f = part_factor(s_ml[w][h][0], s_ml[w][h][1], m);
            l += f * s_ml[w][h][1];
            add_scaled(x, f, *reinterpret_cast<const float4*>(so + (w * NH + h) * HD + d));
        }
        *reinterpret_cast<float4*>(so + h * HD + d) = x;      // warp 0's place of these very numbers: nobody else reads it
        if (d == 0) { s_cta[h][0] = m; s_cta[h][1] = l; }
    }
    const unsigned C = cluster_size(), rank = cluster_rank();
    if (C > 1) cluster_sync(); else __syncthreads();
    const int range = blockIdx.x / C;
    auto put = [&](int h, int d, const float4& x, float m, float l) {
        const int64_t at = (int64_t)token * a.n_heads + head0 + h;
        if (a.ranges == 1) {
            store_row4(reinterpret_cast<T*>(a.out) + at * HD + d, x, l);
        } else {
            *reinterpret_cast<float4*>(a.part_o + (at * a.ranges + range) * HD + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (at * a.ranges + range) * 2) = make_float2(m, l);
        }
    };
    if (C == 1) {
        for (int u = tid; u < nh * (HD / 4); u += DEC_WARPS * 32) {
            const int h = u / (HD / 4), d = (u - h * (HD / 4)) * 4;
            put(h, d, *reinterpret_cast<const float4*>(so + h * HD + d), s_cta[h][0], s_cta[h][1]);
        }
        return;
    }
    // All that is read of the others is read before the arrival, and stored behind it: a CTA leaves when the others have what they read of
    // it, without waiting for its rows to be stored (one arrival behind the stores: 2400 cycles of a call of 10700).
    constexpr int SHARE = (NH * (HD / 4) + 2 * DEC_WARPS * 32 - 1) / (2 * DEC_WARPS * 32);       // of a thread, in clusters of two
    float4 x[SHARE];
    float m[SHARE], l[SHARE];
#pragma unroll
    for (int i = 0; i < SHARE; i++) {
        const int u = (i * (int)C + (int)rank) * DEC_WARPS * 32 + tid, h = u / (HD / 4), d = (u - h * (HD / 4)) * 4;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        m[i] = -INFINITY;
        l[i] = 0.f;
        if (u >= nh * (HD / 4)) continue;
        float2 ml[8];
        float4 px[8];
#pragma unroll
        for (unsigned c = 0; c < 8; c++) {
            ml[c] = make_float2(-INFINITY, 0.f);
            px[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < C) {
                ml[c] = peer_load2(&s_cta[h][0], c);
                px[c] = peer_load4(so + h * HD + d, c);
            }
        }
#pragma unroll
        for (unsigned c = 0; c < 8; c++) m[i] = fmaxf(m[i], ml[c].x);
#pragma unroll
        for (unsigned c = 0; c < 8; c++) {
            const float f = part_factor(ml[c].x, ml[c].y, m[i]);
            l[i] += f * ml[c].y;
            add_scaled(x[i], f, px[c]);
        }
    }
    cluster_arrive();
#pragma unroll
    for (int i = 0; i < SHARE; i++) {
        const int u = (i * (int)C + (int)rank) * DEC_WARPS * 32 + tid, h = u / (HD / 4), d = (u - h * (HD / 4)) * 4;
        if (u < nh * (HD / 4)) put(h, d, x[i], m[i], l[i]);
    }
    cluster_wait();
}

template <typename T, int NG, int SPREAD = 0>
int launch_decode(const DecodeArgs& a, int n_tokens, int cluster, cudaStream_t stream) {
    constexpr size_t smem = DecodeShape<T, NG, SPREAD>::SMEM;
    static_assert(smem <= 227 * 1024, "shared memory");
    auto kernel = attn_decode_q8_kernel<T, NG, SPREAD>;
    static std::atomic<uint64_t> opened{0};                           // devices on which the kernel may have its shared memory
    cudaError_t e = smem > 48 * 1024 ? open_shared_memory((const void*)kernel, (int)smem, opened) : cudaSuccess;
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
        launch_join<T, HD>(a.out, a.part_o, a.part_ml, a.ranges, a.n_heads, (int64_t)n_tokens * a.n_heads, nullptr, 0, stream);
    }
    KLLM_LAUNCH_STATUS();
}

// ---- portions of prompts -------------------------------------------------------------------------------------------------
//
// A CTA takes 64 rows = (tokens of one request's portion) x (heads of one kv group), 16 a warp, and walks the portion's keys
// in tiles of 64.  A tile is converted to float16 once, on its way into shared memory, and read from there by all warps
// as operands (ldmatrix); the next tile's bytes are in registers meanwhile.  Weights go from the first product's result to
// the second's operand in registers.
//
// This form serves float32 and the head sizes that attention_q8_tcgen05.cu does not; its products are bound by mma.sync and by the
// chain of a warp's 16 rows.  Measured, one prompt alone, back to back: float32, 2048 tokens of 32 heads over 4 of 64 172 us (100 TFLOP/s
// counted once; the parts make three products and two of every one), over 8 of 128 310 us (111); 333 tokens 23.4 us (six tiles one
// behind the other); bfloat16, 2048 tokens of 24 heads over 8 of 96 114 us (170), 16 over 8 of 256 222 us (155).

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

// CTAs an SM that there are registers for: with two at head size 64, 2048 float32 tokens of 32 heads over 4 took 195 us for 172.
constexpr int PRE_CTAS = HD <= 32 ? 4 : HD <= 96 ? 3 : 2;

template <typename T>
__global__ void __launch_bounds__(PRE_THREADS, PRE_CTAS) attn_prefill_q8_kernel(const PrefillArgs a) {
    constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
    constexpr int LOADS = PRE_KEYS * PIECES / PRE_THREADS;   // pieces of K (and of V) a thread carries
    static_assert(PRE_KEYS * PIECES % PRE_THREADS == 0, "pieces per thread");
    extern __shared__ __align__(128) unsigned char smem[];
    __half* sq = reinterpret_cast<__half*>(smem);                     // [NQ][rows][PRE_LD]
    __half* sk = sq + NQ * PRE_ROWS * PRE_LD;                         // [keys][PRE_LD]
    __half* sv = sk + PRE_KEYS * PRE_LD;
    __shared__ float s_mul[PRE_KEYS], s_ev[PRE_KEYS], s_inv[PRE_KEYS];   // per key: 2^ek, ev (-inf: not there), 2^-ev
    __shared__ int s_row[PRE_KEYS];
    __shared__ float s_factor[PRE_ROWS];
    __shared__ Portion s_portion;
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x % a.n_kv, gs = a.n_heads / a.n_kv;
    if (warp == 0) {
        Portion p;                                        // longest key ranges first
        if (!find_portion(a.q_start, a.start_pos, a.n_requests, a.tokens_per_tile, (gridDim.x - 1 - blockIdx.x) / a.n_kv, p)) p.req = -1;
        if (lane == 0) s_portion = p;
    }
    __syncthreads();
    const int req = s_portion.req, tok0 = s_portion.tok0, pos0 = s_portion.pos0;
    if (req < 0) return;                                  // the grid is an upper bound on the tiles
    const int n_tok = min(min(a.tokens_per_tile, s_portion.end - tok0), a.n_tokens - tok0);
    if (n_tok <= 0) return;
    const int lo = (a.window > 0 && pos0 >= a.window) ? pos0 - a.window + 1 : 0;
    const int hi = keys_end((int64_t)pos0 + n_tok, a.max_blocks, a.page_size);
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
    float next_k = 1.f, next_v = 1.f;                     // the scales of its page
    auto lookup = [&](int tile) {                         // threads 0..63: one key each
        next_row = -1;
        const int key = tile * PRE_KEYS + tid;
        if (tid >= PRE_KEYS || key < lo || key >= hi) return;
        const int lp = key / a.page_size;
        if (lp >= a.max_blocks) return;
        const int page = table[lp];
        if ((unsigned)page >= (unsigned)a.n_pages) return;
        const int cell = page * a.n_kv + kvh;
        next_row = cell * a.page_size + key - lp * a.page_size;
        next_k = a.kscale[cell];
        next_v = a.vscale[cell];
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
        if (tid < PRE_KEYS) {
            const int e = q8_exponent(next_v);
            s_mul[tid] = q8_pow2(q8_exponent(next_k));
            s_ev[tid] = next_row < 0 ? -INFINITY : (float)e;
            s_inv[tid] = q8_pow2(-e);
        }
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
                if constexpr (NQ == 1) {
                    mma16816(s[2 * n], qa[0][0], qa[0][1], qa[0][2], qa[0][3], b[0], b[1]);
                    mma16816(s[2 * n + 1], qa[0][0], qa[0][1], qa[0][2], qa[0][3], b[2], b[3]);
                } else {
                    // The tensor core cuts its sums; beside float32 queries 16 products at a time are added to a sum in registers (one
                    // sum over 256 dims was four times as far from 64 bits as the single tokens' scores).  It costs 5 to 11 %.
                    float part[2][4];
                    mma16816_first(part[0], qa[NQ - 1][0], qa[NQ - 1][1], qa[NQ - 1][2], qa[NQ - 1][3], b[0], b[1]);
                    mma16816_first(part[1], qa[NQ - 1][0], qa[NQ - 1][1], qa[NQ - 1][2], qa[NQ - 1][3], b[2], b[3]);
#pragma unroll
                    for (int j = NQ - 2; j >= 0; j--) {
                        mma16816(part[0], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b[0], b[1]);
                        mma16816(part[1], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b[2], b[3]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        s[2 * n][j] += part[0][j];
                        s[2 * n + 1][j] += part[1][j];
                    }
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
                    if (key > p_row[i] || (a.window > 0 && p_row[i] - key >= a.window) || ev == -INFINITY) x = -INFINITY;
                    mx[i] = fmaxf(mx[i], x);
                }
            }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            if (mx[i] > moves_above(m_ref[i])) {
                const float corr = m_ref[i] == -INFINITY ? 0.f : exp2f(m_ref[i] - mx[i]);
                m_ref[i] = mx[i];
                l_run[i] *= corr;
#pragma unroll
                for (int n = 0; n < HD / 8; n++) { o[n][2 * i] *= corr; o[n][2 * i + 1] *= corr; }
            }
        }
        float l_tile[2] = {0.f, 0.f};
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
                    l_tile[i] = fmaf(x, inv, l_tile[i]);
                }
            }
        l_run[0] += l_tile[0];
        l_run[1] += l_tile[1];
        uint32_t pa[PRE_KEYS / 16][NP][4];
#pragma unroll
        for (int kk = 0; kk < PRE_KEYS / 16; kk++)
#pragma unroll
            for (int x = 0; x < 4; x++) {                 // a0: row g, keys 2t; a1: row g + 8; a2, a3: keys + 8
                const int n = 2 * kk + (x >> 1), i = x & 1;
                __half h0[NP], h1[NP];
                split<NP>(s[n][2 * i], h0);
                split<NP>(s[n][2 * i + 1], h1);
#pragma unroll
                for (int j = 0; j < NP; j++) {
                    const __half2 hh = __halves2half2(h0[j], h1[j]);
                    pa[kk][j][x] = *reinterpret_cast<const uint32_t*>(&hh);
                }
            }
        // The tensor core cuts its sums: a tile's keys are added to a sum in registers.  One sum over 4000 keys was four times as far from
        // 64 bits as float32 arithmetic, and over 131072 keys a third of half a bfloat16 step (bfloat16, 2048 tokens of 24 heads over 8 of 96: 115 us
        // for 111).
#pragma unroll
        for (int n = 0; n < HD / 16; n++) {
            float part[2][4];
#pragma unroll
            for (int kk = 0; kk < PRE_KEYS / 16; kk++) {
                uint32_t b[4];
                ldmatrix4t(sv_u + vb_off + (unsigned)(kk * 16 * PRE_LD * 2) + n * 32, b);
#pragma unroll
                for (int j = NP - 1; j >= 0; j--) {
                    if (kk == 0 && j == NP - 1) {
                        mma16816_first(part[0], pa[kk][j][0], pa[kk][j][1], pa[kk][j][2], pa[kk][j][3], b[0], b[1]);
                        mma16816_first(part[1], pa[kk][j][0], pa[kk][j][1], pa[kk][j][2], pa[kk][j][3], b[2], b[3]);
                    } else {
                        mma16816(part[0], pa[kk][j][0], pa[kk][j][1], pa[kk][j][2], pa[kk][j][3], b[0], b[1]);
                        mma16816(part[1], pa[kk][j][0], pa[kk][j][1], pa[kk][j][2], pa[kk][j][3], b[2], b[3]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[2 * n][j] += part[0][j];
                o[2 * n + 1][j] += part[1][j];
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
    static std::atomic<uint64_t> opened{0};
    const cudaError_t e = open_shared_memory((const void*)attn_prefill_q8_kernel<T>, (int)smem, opened);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(g_kllm_err, sizeof(g_kllm_err), "attention (8 bits): %zu bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
        return (int)e;
    }
    const int64_t ctas = ((int64_t)a.n_tokens / a.tokens_per_tile + a.n_requests) * a.n_kv;
    if (ctas > 0x7fffffffLL) KLLM_FAIL("attention (8 bits): %lld CTAs", (long long)ctas);
    kllm_launch((attn_prefill_q8_kernel<T>), dim3((unsigned)ctas), dim3(PRE_THREADS), smem, stream, a);
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
    if ((((uintptr_t)kcache | (uintptr_t)vcache) & 15) || ((uintptr_t)out & (dtype == KLLM_F32 ? 15 : 7)))
        KLLM_FAIL("attention (8 bits): the caches must be 16-byte aligned, out to four of its numbers");
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
                 window > 0 ? window : 0, ranges,
                 !(q_stride & 3) && !((uintptr_t)q & (dtype == KLLM_F32 ? 15 : 7)), scale};
    const cudaStream_t s = (cudaStream_t)stream;
    if constexpr (HD <= 128) {
        if (a.heads_per_cta > 8)
            return dtype == KLLM_F32 ? launch_decode<float, 2>(a, n_tokens, cluster, s) : launch_decode<bf16, 2>(a, n_tokens, cluster, s);
    }
    if (dtype == KLLM_F32 && a.heads_per_cta <= 2) return launch_decode<float, 1, 2>(a, n_tokens, cluster, s);
    if (dtype == KLLM_F32 && a.heads_per_cta <= 4) return launch_decode<float, 1, 4>(a, n_tokens, cluster, s);
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
extern "C" int kllm_attention_decode_q8_packed(const void* args) { return call_packed(&kllm_attention_decode_q8, args); }
extern "C" int kllm_attention_prefill_q8_packed(const void* args) { return call_packed(&kllm_attention_prefill_q8, args); }
