// Causal grouped-query attention of prompt portions over the paged cache in 8 bits (q8.cuh) on the fifth-generation tensor
// cores: bfloat16 queries, head size 64 or 128 (-DKLLM_HD).  The mathematics is that of attention_q8.cu; both products
// are float16 tcgen05.mma instructions with float32 accumulators in tensor memory (TMEM).
//
// What bounds it: per 128 x 128 scores of head size 128 the tensor core needs 1024 cycles, the exponentials (16 a cycle and SM)
// as many, and shared memory, from which the products read their operands, nearly so.  So keys and values are converted
// to float16 once for as many rows as fit: a CTA takes two tiles of 128 rows = (tokens of one request's portion) x (heads of
// one kv group), TMEM's 512 columns hold both tiles' scores and outputs, and it walks the keys in tiles of 128.  While the
// softmax of one row tile runs, the tensor core works on the other.  Roles, which meet only at mbarriers:
//
//   warps 0-3, 4-7   softmax of the first and second row tile: a thread owns a row (a TMEM lane).  It brings its queries into
//                    shared memory as float16 (divided by a power of two), then per step reads its 128 scores, applies mask and
//                    online softmax, and writes the weights as float16 over the scores; the second product reads
//                    its A operand from there.
//   warps 8-11, 12-15  loaders of keys and of values: a tile's bytes from the pages into registers a step ahead, converted to float16 and stored in the
//                    128-byte-swizzled layout that the descriptors name (panels of 64 dims, 8-row groups of 1024 bytes,
//                    the 16-byte piece index XORed with the row index modulo 8).
//   warp 16          issues every tcgen05.mma, one elected thread.
//   warp 17          planner: a few steps ahead of the loader, the rows of a tile's keys and their pages' scales.
//
// Scales.  Within a tile's step all keys share one exponent eK and one eV: the loader multiplies every key row by
// 2^(ek - eK) and every value row by 2^(ev - eV) as it converts, exactly, as long as the difference is within +-7
// (448 * 2^7 and 2^-9 * 2^-7 are float16 numbers).  It takes the exponents of the tile's first key for eK and eV; keys whose
// pages differ by more wait for a further step over the same tile, in which they are the ones that are seen (page scales of
// one tile are hardly ever so far apart).  So a step has one factor for its scores, one shift for its weights and one
// for the sum, none of them per score.
//
// The output accumulates in TMEM; a row's reference is moved only when its maximum has grown by more than 2^7.875 (then the row of the
// accumulator is read, rescaled and written back between two products).  Few row tiles behind a long context are cut
// over the keys: every part leaves its unscaled rows, references and sums, which a second kernel joins in order.
//
// Measured, back to back: one prompt of 8192 tokens, 32 heads over 4 of 64: 423 us (650 TFLOP/s), over 8 of 128: 565 us (973, 58 % of a
// library product's 1671); 2048 tokens: 39.6 and 54 us; 512 behind 7680 over 8 of 128: 89 us.  A step of two row tiles takes 4300 cycles at
// head size 128 (3300 at 64), of which the tensor core is busy for 2048 (1024) and the exponentials for 2048: a row tile's own chain of
// scores, maximum, exponentials (1700, at 16 a cycle 1024 alone) and product bounds it, with two softmax warps a scheduler to
// interleave.  Slower: two threads a row (8192 tokens, head size 64: 525 us against 419), a cubic for some of the exponentials (446 to
// 518), loads of scores overlapped with their maximum (428), weights handed over whole at head size 128 (652 against 620).
//
// Every wait on an mbarrier is bounded by a cycle count: a wait that runs out raises a flag in shared memory and sets the
// status word, every role leaves its loop, and the CTA frees its TMEM and returns.
#include "q8.cuh"

#include <limits.h>

#ifndef KLLM_HD
#error "compile with -DKLLM_HD=64 or 128"
#endif

KLLM_EXPORT_LAST_ERROR(attention_q8_tcgen05)

#include "tc5_common.cuh"

namespace {

constexpr int HD = KLLM_HD;
static_assert(HD == 64 || HD == 128, "head size 64 or 128");
constexpr int PANELS = HD / 64;            // 64-dim panels of a row
constexpr int ROWS = 128;                  // query rows of a tile = TMEM lanes
constexpr int TILE = 128;                  // keys of a tile
constexpr int LOADERS = 128;               // threads that bring keys, and as many that bring values
constexpr int THREADS = 640;
constexpr int PANEL = 128 * 128;           // bytes of a panel: 128 rows of 64 float16
constexpr int Q_BYTES = PANELS * PANEL;    // per row tile
constexpr int KV_BYTES = PANELS * PANEL;   // keys or values of a tile
constexpr int STAGES = HD == 64 ? 3 : 2;
constexpr int SBUFS = HD == 64 ? 3 : 2;    // score buffers in TMEM, 128 columns each: taken in turn by the row tiles' steps
constexpr int PARTS = SBUFS == 2 ? 2 : 1;   // parts in which a job's weights are handed over: where the next scores wait for its product
constexpr int PLANS = 4;                   // steps that the planner is ahead of the loader
constexpr int NOTES = 16;                  // steps described at a time; see Note
constexpr int SMEM_BYTES = 1024 + 2 * Q_BYTES + STAGES * 2 * KV_BYTES;
static_assert(SMEM_BYTES <= 226 * 1024, "shared memory");
constexpr unsigned COL_S = 0, COL_O = SBUFS * TILE;      // scores / weights, outputs of the row tiles (HD columns each)
constexpr int TMEM_COLS = 512;
static_assert(SBUFS * TILE + 2 * HD <= TMEM_COLS, "tensor memory");
constexpr int REGS_SOFTMAX = 168, REGS_LOADER = 48, REGS_ISSUER = 48;
// setmaxnreg moves registers inside the CTA's own allocation (threads x registers at launch, multiples of 8)
static_assert(2 * REGS_SOFTMAX + 2 * REGS_LOADER + REGS_ISSUER <= THREADS / 128 * (65536 / THREADS / 8 * 8), "setmaxnreg budget");
static_assert(PLANS + STAGES < NOTES, "notes");
constexpr int PIECES = HD / 16;            // 16-byte pieces of a stored row
constexpr int LOADS = TILE * PIECES / LOADERS;           // pieces of the keys (of the values) a loader thread carries
constexpr int KEY_STEP = LOADERS / PIECES;               // its pieces' keys are so far apart
constexpr int ROW_LANES = HD / 8, ROWS_AT_ONCE = 32 / ROW_LANES;   // rows of 16-bit numbers as a warp reads and writes them
constexpr float kLoud = 262144.f;          // from 2^18 on float32 numbers are 2^-5 and more apart
constexpr int E_SPAN = 7;                  // how far a key's exponents may be from its step's

// What the planner says of a step to everybody.  The note of step t is written once the values of step t - PLANS are converted,
// for which the products of step t - PLANS - STAGES are through: nobody still reads a note of an earlier step.
struct Note {
    int key0, ek, ev, last;
    uint32_t member[4];                    // the keys of the tile that this step is for
};
// ... and to the loader: the keys' rows in the stores, and what they are multiplied with (2^difference as two float16; 0: not of
// this step).
struct __align__(16) Plan {               // read and written four words at a time
    int row[TILE];
    uint32_t kmul[TILE], vmul[TILE];
};

// Instruction descriptor: float32 accumulator, float16 A and B, M x N, B optionally MN-major.
__host__ __device__ constexpr uint32_t make_idesc_f16(int m, int n, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2), descriptor version 1, in two words.  K-major operands:
// 8-row groups 1024 bytes apart (stride offset), leading offset 1.  MN-major operands: 8-k groups 1024 bytes apart (stride
// offset), 64-element panels `lbo_bytes` apart (leading offset).
__device__ __forceinline__ uint32_t desc_lo(unsigned addr, unsigned lbo_bytes) {
    return ((addr >> 4) & 0x3FFFu) | (((lbo_bytes >> 4) & 0x3FFFu) << 16);
}
__host__ __device__ constexpr uint32_t desc_hi(unsigned sbo_bytes) {
    return ((sbo_bytes >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);
}
__device__ __forceinline__ void umma_words(unsigned d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 da, {%1, %3};\nmov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}\n"
                 ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi(1024)), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
__device__ __forceinline__ void umma_tmem_a_words(unsigned d_tmem, unsigned a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(desc_hi(1024)), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
// shared-memory writes of this thread become visible to the tensor core's (async proxy) reads
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// byte offset of 16-byte chunk `ch` (0..7) of row `r` inside a swizzled panel of 128-byte rows
__device__ __forceinline__ unsigned swz(int r, int ch) {
    return (unsigned)((r >> 3) * 1024 + (r & 7) * 128 + ((ch ^ (r & 7)) << 4));
}
__device__ __forceinline__ void tmem_ld8(unsigned taddr, float (&v)[8]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st8(unsigned taddr, const float (&v)[8]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void store16(unsigned addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16 bytes, or as many zeros
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint4 load_shared16(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t half2_times(uint32_t x, uint32_t m) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(x), "r"(m));
    return r;
}
// two float32 at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// mbar_wait and mbar_arrive of tc5_common.cuh by 32-bit shared addresses: a generic pointer is two registers, and the roles
// here have none to spare
__device__ __forceinline__ bool try_at(unsigned bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_at(unsigned bar, unsigned parity, unsigned abort_at, int* status, int where) {
    if (try_at(bar, parity)) return true;
    const long long t0 = clock64();
    unsigned spins = 0;
    while (!try_at(bar, parity)) {
        if ((++spins & 255u) == 0) {
            int gone;
            asm volatile("ld.volatile.shared.b32 %0, [%1];\n" : "=r"(gone) : "r"(abort_at) : "memory");
            if (gone) return false;
            if (clock64() - t0 > kCycleLimit) {
                asm volatile("st.volatile.shared.b32 [%0], %1;\n" ::"r"(abort_at), "r"(1) : "memory");
                if (status) atomicCAS(status, 0, where);
                return false;
            }
        }
    }
    return true;
}
__device__ __forceinline__ bool wait_warp_at(unsigned bar, unsigned parity, unsigned abort_at, int* status, int where) {
    return __all_sync(0xffffffffu, wait_at(bar, parity, abort_at, status, where));
}
__device__ __forceinline__ void arrive_at(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ uint32_t word_at(unsigned addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// What a CTA is about, worked out by one thread.  Every role reads what it needs of it from shared memory: values that all roles
// derive from registers are kept, or spilled, for all of them.
struct Work {
    int req, tok0, n_tok, tiles, pos0, lo, hi, tile_lo, tile_hi;     // request (-1: none), rows, row tiles in use, keys, tiles of keys
};

struct Args {
    bf16* out;
    float* part_o;               // [n, heads, splits, HD], part_ml [n, heads, splits, 2]: NULL with one
    float* part_ml;
    const bf16* q;
    int64_t q_stride;
    const uint8_t* kcache;
    const uint8_t* vcache;
    const float* kscale;
    const float* vscale;
    const int* q_start;
    const int* start_pos;
    const int* block_table;
    int max_blocks, n_pages, n_tokens, n_requests, n_heads, n_kv, page_size, window, tokens_per_tile, row_tiles, splits;
    bool q_by_eight;             // rows of queries may be read 16 bytes at a time
    float scale;
    int* status;
};

__global__ void __launch_bounds__(THREADS, 1) attn_prefill_q8_tc5_kernel(const Args a) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bar_k_full[STAGES], bar_k_empty[STAGES], bar_v_full[STAGES], bar_v_empty[STAGES];
    __shared__ __align__(8) uint64_t bar_q_full[2], bar_s_full[SBUFS], bar_p_full[SBUFS][PARTS], bar_pv[2], bar_note[NOTES];
    __shared__ __align__(8) uint64_t bar_plan_full[PLANS], bar_plan_empty[PLANS];
    __shared__ Note s_note[NOTES];
    __shared__ Plan s_plan[PLANS];
    static_assert(alignof(Plan) == 16 && sizeof(Plan) % 16 == 0, "four words at a time");
    __shared__ unsigned s_tmem;
    __shared__ volatile Work s_work;
    __shared__ int s_abort;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    griddep_wait();
    griddep_launch();
    if (warp == 0) {
        // CTAs start in the order of blockIdx.x: longest key ranges first, all kv heads and parts of a range side by side
        const int per_cta = a.tokens_per_tile * a.row_tiles, split = blockIdx.x % a.splits;
        Portion p;
        if (!find_portion(a.q_start, a.start_pos, a.n_requests, per_cta, (gridDim.x - 1 - blockIdx.x) / (a.n_kv * a.splits), p)) p.req = -1;
        const int tok0 = p.tok0, pos0 = p.pos0, n_tok = p.req >= 0 ? min(per_cta, min(p.end, a.n_tokens) - tok0) : 0;
        if (lane == 0) s_work.req = n_tok > 0 ? p.req : -1;
        if (lane == 0 && n_tok > 0) {
            const int hi = max(keys_end((int64_t)pos0 + n_tok, a.max_blocks, a.page_size), 1);
            // one tile at least: every role takes at least one step (a window behind the table's end sees nothing in it)
            const int lo = min((a.window > 0 && pos0 >= a.window) ? pos0 - a.window + 1 : 0, hi - 1);
            // this part's tiles of keys; a part without any leaves zeros
            const int first = lo / TILE, all = (hi + TILE - 1) / TILE - first, per = (all + a.splits - 1) / a.splits;
            s_work.tok0 = tok0;
            s_work.n_tok = n_tok;
            s_work.tiles = n_tok > a.tokens_per_tile ? 2 : 1;
            s_work.pos0 = pos0;
            s_work.lo = lo;
            s_work.hi = hi;
            s_work.tile_lo = first + min(all, split * per);
            s_work.tile_hi = first + min(all, (split + 1) * per);
        }
    }
    if (threadIdx.x == 32) {
        s_abort = 0;
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&bar_k_full[i], LOADERS); mbar_init(&bar_k_empty[i], 1);
            mbar_init(&bar_v_full[i], LOADERS); mbar_init(&bar_v_empty[i], 1);
        }
        for (int i = 0; i < SBUFS; i++) {
            mbar_init(&bar_s_full[i], 1);
            for (int j = 0; j < PARTS; j++) mbar_init(&bar_p_full[i][j], ROWS);
        }
        for (int i = 0; i < 2; i++) { mbar_init(&bar_q_full[i], ROWS); mbar_init(&bar_pv[i], 1); }
        for (int i = 0; i < NOTES; i++) mbar_init(&bar_note[i], 32);
        for (int i = 0; i < PLANS; i++) { mbar_init(&bar_plan_full[i], 32); mbar_init(&bar_plan_empty[i], 2 * LOADERS); }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    volatile unsigned* tmem_at = &s_tmem;
    if (s_work.req < 0) {                      // the grid is an upper bound on the tiles
        if (warp == 16)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(__shfl_sync(0xffffffffu, *tmem_at, 0)), "r"(TMEM_COLS));
        return;
    }
    const unsigned abort_at = smem_u32(&s_abort);
    const bool nothing = s_work.tile_lo >= s_work.tile_hi;
    // swizzled tiles want 1024-byte alignment
    auto shared_base = [&]() { return (smem_u32(smem_raw) + 1023u) & ~1023u; };

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_ISSUER));
        if (warp == 16 && !nothing) {
            // ---- the issuer.  A job is a row tile's step; jobs go round the score buffers.  The scores of the first SBUFS jobs,
            // then for every job weights x values and the scores of the job SBUFS behind it, whose buffer that product has read
            // (the tensor core works in the order of issue).
            const int tiles = s_work.tiles;
            const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_at, 0), sQ = shared_base(), sK = sQ + 2 * Q_BYTES, sV = sK + STAGES * KV_BYTES;
            constexpr uint32_t IDESC_S = make_idesc_f16(ROWS, TILE, false), IDESC_O = make_idesc_f16(ROWS, HD, true);
            const uint32_t q_lo0 = desc_lo(sQ, 16), k_lo0 = desc_lo(sK, 16), v_lo0 = desc_lo(sV, PANEL);
            int s_step = 0, s_x = 0, s_buf = 0, ks = 0;        // the next scores: step, row tile, buffer; stage of its keys
            unsigned kp = 0;
            int last_step = INT_MAX;                           // known once its scores are issued
            bool s_done = false;
            auto next_scores = [&]() -> bool {
                if (s_done) return true;
                if (s_x == 0) {
                    if (!wait_warp_at(smem_u32(&bar_k_full[ks]), kp, abort_at, a.status, 3)) return false;
                    // the loader that announces the keys has seen the planner's note
                    if (s_note[s_step % NOTES].last) last_step = s_step;
                }
                if (s_step == 0 && !wait_warp_at(smem_u32(&bar_q_full[s_x]), 0, abort_at, a.status, 2)) return false;
                fence_async_smem();
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t q_lo = q_lo0 + (uint32_t)(s_x * (Q_BYTES >> 4)), k_lo = k_lo0 + (uint32_t)(ks * (KV_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t off = (uint32_t)(((kk >> 2) * PANEL + (kk & 3) * 32) >> 4);
                        umma_words(tmem + COL_S + s_buf * TILE, q_lo + off, k_lo + off, IDESC_S, kk > 0);
                    }
                    umma_commit(&bar_s_full[s_buf]);
                    if (s_x == tiles - 1) umma_commit(&bar_k_empty[ks]);
                }
                __syncwarp();
                s_buf = s_buf + 1 == SBUFS ? 0 : s_buf + 1;
                if (++s_x == tiles) {
                    s_x = 0;
                    s_step++;
                    s_done = s_step > last_step;
                    if (++ks == STAGES) { ks = 0; kp ^= 1u; }
                }
                return true;
            };
            bool ok = true;
            for (int i = 0; ok && i < SBUFS; i++) ok = next_scores();
            int step = 0, x = 0, buf = 0, vs = 0;              // of the next product
            unsigned pp = 0, vp = 0;
            while (ok) {
                if (x == 0) ok = wait_warp_at(smem_u32(&bar_v_full[vs]), vp, abort_at, a.status, 4);
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    // these weights are in tensor memory, and the output is rescaled
                    ok = ok && wait_warp_at(smem_u32(&bar_p_full[buf][part]), pp, abort_at, a.status, 5);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t v_lo = v_lo0 + (uint32_t)(vs * (KV_BYTES >> 4));
#pragma unroll
                        for (int kk = part * (TILE / 16 / PARTS); kk < (part + 1) * (TILE / 16 / PARTS); kk++)
                            umma_tmem_a_words(tmem + COL_O + x * HD, tmem + COL_S + buf * TILE + (unsigned)(kk * 8),
                                              v_lo + (uint32_t)(kk * (2048 >> 4)), IDESC_O, step > 0 || kk > 0);
                        if (part == PARTS - 1) {
                            umma_commit(&bar_pv[x]);
                            if (x == tiles - 1) umma_commit(&bar_v_empty[vs]);
                        }
                    }
                    __syncwarp();
                }
                ok = ok && next_scores();
                if (!ok || (step == last_step && x == tiles - 1)) break;
                if (++buf == SBUFS) { buf = 0; pp ^= 1u; }
                if (++x == tiles) {
                    x = 0;
                    step++;
                    if (++vs == STAGES) { vs = 0; vp ^= 1u; }
                }
            }
        }
        if (warp == 17 && !nothing) {
            // ---- the planner: which keys a step is for, where they lie, what they are multiplied with.  A lane looks after four
            // neighbouring keys of a tile.  Where these lie in one page (page sizes in steps of four) pages are read two tiles
            // ahead of their step, scales one; otherwise each when it is needed.
            const int lo = s_work.lo, hi = s_work.hi, tile_hi = s_work.tile_hi, kvh = (blockIdx.x / a.splits) % a.n_kv;
            const int* table = a.block_table + (int64_t)s_work.req * a.max_blocks;
            const bool quads = a.page_size % 4 == 0;
            int page = -1, first_row = -1;
            float ksc = 1.f, vsc = 1.f;
            auto page_of = [&](int key) {
                const int lp = key / a.page_size;
                return key < hi && lp < a.max_blocks ? load_early(table + lp) : -1;
            };
            auto place = [&](int pg, int key) {
                first_row = -1;
                if ((unsigned)pg >= (unsigned)a.n_pages) return;
                const int cell = pg * a.n_kv + kvh;
                first_row = cell * a.page_size + key % a.page_size;
                ksc = load_early(a.kscale + cell);
                vsc = load_early(a.vscale + cell);
            };
            auto exponents = [&]() { return (q8_exponent(ksc) << 16) | (q8_exponent(vsc) & 0xffff); };
            int key = s_work.tile_lo * TILE + lane * 4;        // the lane's first
            if (quads) {
                place(page_of(key), key);
                page = page_of(key + TILE);
            }
            bool ok = true;
            int step = 0;
#pragma unroll 1
            for (int tile = s_work.tile_lo; ok && tile < tile_hi; tile++, key += TILE) {
                int at[4], exps[4];                            // rows in the stores, exponents of the scales (INT_MIN: no key)
                if (quads) {
                    const int e = exponents();
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool there = first_row >= 0 && key + i >= lo && key + i < hi;
                        at[i] = there ? first_row + i : -1;
                        exps[i] = there ? e : INT_MIN;
                    }
                    place(page, key + TILE);
                    page = page_of(key + 2 * TILE);
                } else {
#pragma unroll 1
                    for (int i = 0; i < 4; i++) {
                        place(key + i >= lo ? page_of(key + i) : -1, key + i);
                        const int r = first_row, e = r < 0 ? INT_MIN : exponents();
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (j == i) { at[j] = r; exps[j] = e; }
                    }
                }
                bool done = false;
#pragma unroll 1
                while (ok && !done) {
                    // the first key that is left names the step's exponents; those near enough join it
                    const int mine = exps[0] != INT_MIN ? exps[0] : exps[1] != INT_MIN ? exps[1] : exps[2] != INT_MIN ? exps[2] : exps[3];
                    const unsigned have = __ballot_sync(0xffffffffu, mine != INT_MIN);
                    const int lead = have ? __shfl_sync(0xffffffffu, mine, __ffs(have) - 1) : 0;
                    const int ek = lead >> 16, ev = (int)(short)(lead & 0xffff);
                    uint32_t kmul[4], vmul[4], bits = 0;
                    bool left = false;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int dk = (exps[i] >> 16) - ek, dv = (int)(short)(exps[i] & 0xffff) - ev;
                        const bool in = exps[i] != INT_MIN && abs(dk) <= E_SPAN && abs(dv) <= E_SPAN;
                        kmul[i] = in ? (uint32_t)(dk + 15) * 0x04000400u : 0u;
                        vmul[i] = in ? (uint32_t)(dv + 15) * 0x04000400u : 0u;
                        if (in) { bits |= 1u << i; exps[i] = INT_MIN; }
                        left = left || exps[i] != INT_MIN;
                    }
                    done = !__any_sync(0xffffffffu, left);
                    // eight lanes' four bits are a word
                    uint32_t word = bits << ((lane & 7) * 4);
#pragma unroll
                    for (int d = 1; d < 8; d <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, d);
                    const int p = step % PLANS;
                    ok = wait_warp_at(smem_u32(&bar_plan_empty[p]), ((unsigned)(step / PLANS) & 1u) ^ 1u, abort_at, a.status, 12);
                    if (!ok) break;
                    Note& note = s_note[step % NOTES];
                    if ((lane & 7) == 0) note.member[lane >> 3] = word;
                    if (lane == 0) { note.key0 = tile * TILE; note.ek = ek; note.ev = ev; note.last = done && tile + 1 == tile_hi; }
                    *reinterpret_cast<int4*>(&s_plan[p].row[lane * 4]) = make_int4(at[0], at[1], at[2], at[3]);
                    *reinterpret_cast<uint4*>(&s_plan[p].kmul[lane * 4]) = make_uint4(kmul[0], kmul[1], kmul[2], kmul[3]);
                    *reinterpret_cast<uint4*>(&s_plan[p].vmul[lane * 4]) = make_uint4(vmul[0], vmul[1], vmul[2], vmul[3]);
                    arrive_at(smem_u32(&bar_note[step % NOTES]));
                    arrive_at(smem_u32(&bar_plan_full[p]));
                    step++;
                }
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_LOADER));
        // ---- loaders, one group for the keys and one for the values: a step's bytes into registers while the step before is
        // being used, converted in pairs, float16 into the stages
        if (!nothing) {
            const bool values = warp >= 12;
            const int tid = threadIdx.x & 127;
            const unsigned stages = shared_base() + 2 * Q_BYTES + (values ? STAGES * KV_BYTES : 0);
            const uint8_t* store = values ? a.vcache : a.kcache;
            const unsigned full = smem_u32(values ? bar_v_full : bar_k_full), empty = smem_u32(values ? bar_v_empty : bar_k_empty);
            // a thread's pieces are of keys KEY_STEP apart
            const int piece = tid % PIECES, key_off = tid / PIECES;
            const bool odd_first = PIECES == 8 && piece >= 4;  // the panels of a row at a time on different banks
            const unsigned place = (unsigned)((piece >> 2) * PANEL) + swz(key_off, (piece & 3) * 2 + (odd_first ? 1 : 0));
            store += piece * 16;
            const unsigned rows_at = smem_u32(s_plan[0].row) + key_off * 4;
            const unsigned mul_at = smem_u32(values ? s_plan[0].vmul : s_plan[0].kmul) + key_off * 4;
            uint4 raw[LOADS];
            auto fetch = [&](int p) {
#pragma unroll
                for (int i = 0; i < LOADS; i++) {
                    // where there is no key: the first row, which the conversion leaves out
                    const int r = max((int)word_at(rows_at + p * (unsigned)sizeof(Plan) + i * KEY_STEP * 4), 0);
                    raw[i] = load_early(reinterpret_cast<const uint4*>(store + (int64_t)r * HD));
                }
            };
            int stage = 0;
            unsigned parity = 1;                               // of the stages' "empty" barriers: free at first
            bool ok = wait_at(smem_u32(&bar_plan_full[0]), 0, abort_at, a.status, 1);
            if (ok) fetch(0);
#pragma unroll 1
            for (int step = 0; ok; step++) {
                const int p = step % PLANS, p2 = (step + 1) % PLANS;
                const Note& note = s_note[step % NOTES];
                const bool last = note.last != 0;
                // not all keys of the tile are of this step: the multiplier of the others is 0, and their bytes (which may be
                // NaN) become zeros
                const bool some = (note.member[0] & note.member[1] & note.member[2] & note.member[3]) != 0xffffffffu;
                ok = wait_at(empty + stage * 8, parity, abort_at, a.status, 7);
                if (!ok) break;
                const unsigned dst = stages + stage * KV_BYTES + place;
#pragma unroll
                for (int i = 0; i < LOADS; i++) {
                    const uint32_t m = word_at(mul_at + p * (unsigned)sizeof(Plan) + i * KEY_STEP * 4);
                    uint4 x = raw[i];
                    if (some) {
                        const uint32_t keep = m ? 0xffffffffu : 0u;
                        x.x &= keep; x.y &= keep; x.z &= keep; x.w &= keep;
                    }
                    uint32_t h[8];
                    q8_to_f16x4(x.x, h[0], h[1]); q8_to_f16x4(x.y, h[2], h[3]);
                    q8_to_f16x4(x.z, h[4], h[5]); q8_to_f16x4(x.w, h[6], h[7]);
#pragma unroll
                    for (int j = 0; j < 8; j++) h[j] = half2_times(h[j], m);
                    // rows KEY_STEP apart are whole groups of eight apart: the same place in a later group; the other half of the
                    // piece is the neighbouring chunk, one bit away
                    const unsigned at = dst + (unsigned)(i * KEY_STEP * 128);
                    static_assert(KEY_STEP % 8 == 0, "groups of eight rows");
                    if (odd_first) {
                        store16(at, h[4], h[5], h[6], h[7]);
                        store16(at ^ 16u, h[0], h[1], h[2], h[3]);
                    } else {
                        store16(at, h[0], h[1], h[2], h[3]);
                        store16(at ^ 16u, h[4], h[5], h[6], h[7]);
                    }
                }
                fence_async_smem();
                arrive_at(full + stage * 8);
                arrive_at(smem_u32(&bar_plan_empty[p]));
                if (last) break;
                ok = wait_at(smem_u32(&bar_plan_full[p2]), (unsigned)((step + 1) / PLANS) & 1u, abort_at, a.status, 1);
                if (!ok) break;
                fetch(p2);
                if (++stage == STAGES) { stage = 0; parity ^= 1u; }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS_SOFTMAX));
        // ---- softmax: this thread's row is (token, head of the group) of row tile x -----------------------
        const int gs = a.n_heads / a.n_kv, tpt = a.tokens_per_tile, kvh = (blockIdx.x / a.splits) % a.n_kv, split = blockIdx.x % a.splits;
        const int tok0 = s_work.tok0, n_tok = s_work.n_tok, pos0 = s_work.pos0, tiles = s_work.tiles;
        const unsigned tmem = *tmem_at;
        const int x = warp >> 2, r = threadIdx.x & 127;
        const int tt = x * tpt + r / gs, hh = r % gs;
        const bool valid = r < tpt * gs && tt < n_tok;
        const int p_row = valid ? pos0 + tt : -1;                           // -1: sees no key
        const int w_row = (a.window > 0) ? p_row + 1 - a.window : 0;
        const int64_t at = (int64_t)(tok0 + tt) * a.n_heads + kvh * gs + hh;
        const unsigned lane_base = (unsigned)((warp & 3) * 32) << 16;
        const unsigned t_s0 = tmem + lane_base + COL_S, t_o = tmem + lane_base + COL_O + x * HD;
        float m_ref = -INFINITY, l_run = 0.f;
        bool ok = x < tiles && !nothing;
        if (ok) {
            // the row's queries: float16, its power of two in the factor, the scale's sign in the numbers
            // A warp brings its 32 rows as they are into their places, ROW_LANES lanes a row; then a thread turns its row into float16
            // where it lies.  In short loops: this runs once a CTA, and what is unrolled waits for its instructions to be
            // fetched (16 loads and their shuffles 2200 cycles, the rest 3900 at head size 128).
            const unsigned rows_at = shared_base() + x * Q_BYTES;
            const int64_t own = valid ? (int64_t)(tok0 + tt) * a.q_stride + (int64_t)(kvh * gs + hh) * HD : -1;
            const int piece = lane % ROW_LANES;
#pragma unroll 4
            for (int i = 0; i < ROW_LANES; i++) {
                const int from = i * ROWS_AT_ONCE + lane / ROW_LANES;
                const int64_t off = __shfl_sync(0xffffffffu, own, from);
                const unsigned to = rows_at + (unsigned)((piece >> 3) * PANEL) + swz((warp & 3) * 32 + from, piece & 7);
                const bf16* src = a.q + (off < 0 ? 0 : off) + piece * 8;
                if (a.q_by_eight) {
                    copy16(to, src, off >= 0);
                } else {
                    const unsigned short* h = reinterpret_cast<const unsigned short*>(src);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (off >= 0) v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
                    store16(to, v.x, v.y, v.z, v.w);
                }
            }
            copies_wait();
            __syncwarp();
            uint32_t two = 0;                                                // the row's largest magnitudes at even and odd places
#pragma unroll 4
            for (int c = 0; c < HD / 8; c++) {
                const uint4 v = load_shared16(rows_at + (unsigned)((c >> 3) * PANEL) + swz(r, c & 7));
                two = max_u16x2(two, max_u16x2(max_u16x2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), max_u16x2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
            }
            const int m = (int)max(two << 16, two & 0xffff0000u);
            const bool finite = m < 0x7f800000;
            const float up = finite ? copysignf(q8_pow2(row_shift(m)), a.scale) : 0.f;
#pragma unroll 4
            for (int c = 0; c < HD / 8; c++) {
                const unsigned to = rows_at + (unsigned)((c >> 3) * PANEL) + swz(r, c & 7);
                const uint4 v = load_shared16(to);
                uint32_t h[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (!finite) h[j] = 0;
                    h[j] = q8_half2(__uint_as_float(h[j] << 16) * up, __uint_as_float(h[j] & 0xffff0000u) * up);
                }
                store16(to, h[0], h[1], h[2], h[3]);
            }
            const float factor = finite ? fabsf(a.scale) * kLog2e * q8_pow2(-row_shift(m)) : __int_as_float(0x7fffffff);
            fence_async_smem();
            arrive_at(smem_u32(&bar_q_full[x]));
            bool last = false;
            int step = 0, buf = x % SBUFS;
            unsigned parity = 0;
            // The steps, in the way that is sound for references below 2^18.  False: the scores of `step` are beyond it, and nothing of that
            // step is done.
            auto steps = [&](auto is_loud) -> bool {
            constexpr bool LOUD = decltype(is_loud)::value;
            for (; ok && !last; step++) {
                ok = wait_at(smem_u32(&bar_note[step % NOTES]), (unsigned)(step / NOTES) & 1u, abort_at, a.status, 8) &&
                     wait_at(smem_u32(&bar_s_full[buf]), parity, abort_at, a.status, 9);
                ok = __all_sync(0xffffffffu, ok);             // a warp leaves together, if it does
                if (!ok) break;
                const unsigned t_s = t_s0 + buf * TILE;
                tc_fence_after();
                const Note& note = s_note[step % NOTES];
                last = note.last != 0;
                // never 0 (a scale of 0, tiny queries) nor NaN (queries that are not finite: numbers of 0): -inf has to stay -inf
                const float product = factor * q8_pow2(note.ek), f = product >= 1.1754944e-38f ? product : 1.1754944e-38f;
                const float ev = (float)note.ev, per_sum = q8_pow2(-note.ev);
                // which of the tile's keys this row sees
                const int upto = p_row - note.key0 + 1, from = w_row - note.key0;
                uint32_t seen[4];
                bool masked = false;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    seen[c] = note.member[c] & low_bits(upto - 32 * c) & ~low_bits(from - 32 * c);
                    masked = masked || seen[c] != 0xffffffffu;
                }
                float s[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld32(t_s + c * 32, s[c]);
                tmem_ld_wait();
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!((seen[c] >> j) & 1u)) s[c][j] = -INFINITY;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int j = 0; j < 32; j += 2) mx4[(j >> 1) & 3] = max3(mx4[(j >> 1) & 3], s[c][j], s[c][j + 1]);
                const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                const float mx = top == -INFINITY ? -INFINITY : fmaf(top, f, ev);
                if (!LOUD && __any_sync(0xffffffffu, fabsf(mx) >= kLoud && mx != -INFINITY)) {
                    last = false;
                    return false;
                }
                const bool move = mx > moves_above(m_ref);
                float corr = 1.f;
                if (move) {
                    corr = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
                    m_ref = mx;
                }
                const float ref = m_ref == -INFINITY ? 0.f : m_ref, shift = ev - ref + kLift;
                // The product of this row tile's step before has to be over.  With two score buffers and two row tiles it was
                // issued before these scores, and is; otherwise it is waited for, every time (a wait by parity is only sound for
                // the phase behind the one waited for last).
                if (step > 0) {
                    if (SBUFS != 2 || tiles != 2) {
                        ok = wait_warp_at(smem_u32(&bar_pv[x]), (unsigned)(step - 1) & 1u, abort_at, a.status, 10);
                        if (!ok) break;
                    }
                    if (__any_sync(0xffffffffu, move)) {
                        // rows of this warp rescale what the products so far have added up (rows that did not move multiply by
                        // one); the next product waits for these weights
                        tc_fence_after();
#pragma unroll
                        for (int cb = 0; cb < HD / 8; cb++) {
                            float t[8];
                            tmem_ld8(t_o + cb * 8, t);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 8; j++) t[j] *= corr;
                            tmem_st8(t_o + cb * 8, t);
                        }
                    }
                }
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 f2 = make_float2(f, f), shift2 = make_float2(shift, shift);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float pk[32];
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float2 p = fma2(make_float2(s[half * 2 + c][j], s[half * 2 + c][j + 1]), f2, shift2);
                            if (LOUD) {
                                p.x = fmaf(s[half * 2 + c][j], f, ev) - ref + kLift;
                                p.y = fmaf(s[half * 2 + c][j + 1], f, ev) - ref + kLift;
                            }
                            p.x = fast_exp2(p.x);
                            p.y = fast_exp2(p.y);
                            sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], p);
                            pk[c * 16 + j / 2] = __uint_as_float(q8_half2(p.x, p.y));
                        }
                    tmem_st32(t_s + half * 32, pk);        // over the first 64 columns of the scores
                    if (PARTS == 2 || half == 1) {
                        tmem_st_wait();
                        tc_fence_before();
                        arrive_at(smem_u32(&bar_p_full[buf][PARTS == 2 ? half : 0]));
                    }
                }
                l_run = l_run * corr + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) * per_sum;
                buf += tiles;
                if (buf >= SBUFS) { buf -= SBUFS; parity ^= 1u; }
            }
            return true;
            };
            // Near references so large that float32 numbers are whole units apart, s f + (ev - m_ref) in one rounding puts the largest weight
            // beyond float16: there scores are rounded as the reference was, and then the difference is taken.  A loop of its own, as both
            // in one cost the usual way registers (8192 tokens of head size 128: 597 to 631 us, one more addition a score always 579; this
            // 564, of which the look at the maximum is 5).
            if (!steps(std::false_type{})) steps(std::true_type{});
            if (factor != factor && m_ref != -INFINITY) l_run = factor;        // the row is NaN where it saw a key
            if (ok) ok = wait_warp_at(smem_u32(&bar_pv[x]), (unsigned)(step - 1) & 1u, abort_at, a.status, 11);
            if (ok) {
                tc_fence_after();
                // The rows go through the queries' place in shared memory (their products are through), a warp's 32 by itself, so that
                // neighbouring lanes store neighbouring bytes: 16-byte pieces of a row's 2 HD bytes, XORed with the row as the
                // queries were.  Float32 parts take two passes.
                const unsigned rows_at = shared_base() + x * Q_BYTES + (warp & 3) * 32 * (HD * 2);
                const float inv = a.splits > 1 ? 1.f : l_run == 0.f ? 0.f : 1.f / l_run;
                const int passes = a.splits > 1 ? 2 : 1;
                unsigned char* const rows_out = a.splits > 1 ? reinterpret_cast<unsigned char*>(a.part_o) : reinterpret_cast<unsigned char*>(a.out);
                const int64_t own = a.splits > 1 ? (at * a.splits + split) * (HD * 4) : at * (HD * 2);
#pragma unroll 1
                for (int pass = 0; pass < passes; pass++) {
                    if (a.splits == 1) {
#pragma unroll 1
                        for (int cb = 0; cb < HD / 32; cb++) {
                            float t[32];
                            tmem_ld32(t_o + cb * 32, t);
                            tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                store16(rows_at + lane * (HD * 2) + (((cb * 4 + c) ^ (lane & 7)) << 4),
                                        pack_bf16(t[8 * c] * inv, t[8 * c + 1] * inv), pack_bf16(t[8 * c + 2] * inv, t[8 * c + 3] * inv),
                                        pack_bf16(t[8 * c + 4] * inv, t[8 * c + 5] * inv), pack_bf16(t[8 * c + 6] * inv, t[8 * c + 7] * inv));
                        }
                    } else {
#pragma unroll 1
                        for (int cb = 0; cb < HD / 64; cb++) {
                            float t[32];
                            tmem_ld32(t_o + pass * (HD / 2) + cb * 32, t);
                            tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 8; c++)
                                store16(rows_at + lane * (HD * 2) + (((cb * 8 + c) ^ (lane & 7)) << 4), __float_as_uint(t[4 * c]),
                                        __float_as_uint(t[4 * c + 1]), __float_as_uint(t[4 * c + 2]), __float_as_uint(t[4 * c + 3]));
                        }
                    }
                    __syncwarp();
#pragma unroll 2
                    for (int i = 0; i < ROW_LANES; i++) {
                        const int row = i * ROWS_AT_ONCE + lane / ROW_LANES, piece = lane % ROW_LANES;
                        const int64_t to = __shfl_sync(0xffffffffu, own, row);
                        const bool there = __shfl_sync(0xffffffffu, valid, row);
                        const uint4 v = load_shared16(rows_at + row * (HD * 2) + ((piece ^ (row & 7)) << 4));
                        if (there) *reinterpret_cast<uint4*>(rows_out + to + pass * (HD * 2) + piece * 16) = v;
                    }
                    __syncwarp();
                }
            }
        } else if (valid && nothing) {
            for (int c = 0; c < HD / 4; c++)
                *reinterpret_cast<float4*>(a.part_o + (at * a.splits + split) * HD + 4 * c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (valid && a.splits > 1)
            *reinterpret_cast<float2*>(a.part_ml + (at * a.splits + split) * 2) = make_float2(m_ref, l_run);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(__shfl_sync(0xffffffffu, *tmem_at, 0)), "r"(TMEM_COLS));
}

}  // namespace

extern "C" int kllm_attention_q8_tcgen05_head_dim() { return HD; }

// Requests' portions: rows q_start[s]..q_start[s+1] of request s start at cache position start_pos[s]; bfloat16 rows.  row_tiles:
// tiles of 128 rows a CTA (1 or 2); splits: parts of the keys, with part_o float32 [n, heads, splits, HD] and part_ml
// float32 [n, heads, splits, 2] where there are several.  status: a device int that a bounded wait which ran out sets (1, 7:
// loader, 2-5: issuer, 8-11: softmax, 12: planner).
extern "C" int kllm_attention_prefill_q8_tcgen05(void* out, float* part_o, float* part_ml, const void* q, int64_t q_stride,
                                                 const void* kcache, const void* vcache, const float* kscale,
                                                 const float* vscale, const int* q_start, const int* start_pos,
                                                 const int* block_table, int max_blocks, int n_pages, int n_tokens,
                                                 int n_requests, int n_heads, int n_kv, int hd, int page_size, int window,
                                                 float scale, int row_tiles, int splits, int* status, void* stream) {
    if (n_tokens <= 0 || n_requests <= 0) return 0;
    if (hd != HD) KLLM_FAIL("attention (8 bits, tcgen05): this library was built for head size %d, not %d", HD, hd);
    if (n_kv <= 0 || n_heads <= 0 || n_heads % n_kv) KLLM_FAIL("attention (8 bits, tcgen05): %d heads over %d kv heads", n_heads, n_kv);
    const int gs = n_heads / n_kv;
    if (gs > ROWS) KLLM_FAIL("attention (8 bits, tcgen05): %d heads per kv head, at most %d", gs, ROWS);
    if (page_size <= 0 || n_pages <= 0) KLLM_FAIL("attention (8 bits, tcgen05): %d pages of %d", n_pages, page_size);
    if ((int64_t)n_pages * n_kv * page_size >= (1LL << 31)) KLLM_FAIL("attention (8 bits, tcgen05): a store of 2^31 rows or more");
    if (row_tiles < 1 || row_tiles > 2 || splits < 1) KLLM_FAIL("attention (8 bits, tcgen05): %d row tiles, %d parts", row_tiles, splits);
    if (splits > 1 && (!part_o || !part_ml)) KLLM_FAIL("attention (8 bits, tcgen05): several parts without room for them");
    if (((uintptr_t)out & 15) || (((uintptr_t)kcache | (uintptr_t)vcache) & 15))
        KLLM_FAIL("attention (8 bits, tcgen05): out and the caches must be 16-byte aligned");
    Args a{(bf16*)out, part_o, part_ml, (const bf16*)q, q_stride, (const uint8_t*)kcache, (const uint8_t*)vcache, kscale, vscale,
           q_start, start_pos, block_table, max_blocks, n_pages, n_tokens, n_requests, n_heads, n_kv, page_size,
           window > 0 ? window : 0, ROWS / gs, row_tiles, splits, !((uintptr_t)q & 15) && !(q_stride & 7), scale, status};
    static std::atomic<uint64_t> opened{0};
    const cudaError_t e = open_shared_memory((const void*)attn_prefill_q8_tc5_kernel, SMEM_BYTES, opened);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(g_kllm_err, sizeof(g_kllm_err), "attention (8 bits, tcgen05): %d bytes of shared memory refused: %s", SMEM_BYTES,
                 cudaGetErrorString(e));
        return (int)e;
    }
    const int64_t ctas = ((int64_t)n_tokens / (a.tokens_per_tile * row_tiles) + n_requests) * n_kv * splits;
    if (ctas > 0x7fffffffLL) KLLM_FAIL("attention (8 bits, tcgen05): %lld CTAs", (long long)ctas);
    kllm_launch((attn_prefill_q8_tc5_kernel), dim3((unsigned)ctas), dim3(THREADS), SMEM_BYTES, (cudaStream_t)stream, a);
    if (splits > 1) {
        launch_join<bf16, HD>(out, part_o, part_ml, splits, n_heads, (int64_t)n_tokens * n_heads, q_start, n_requests, (cudaStream_t)stream);
    }
    KLLM_LAUNCH_STATUS();
}
extern "C" int kllm_attention_prefill_q8_tcgen05_packed(const void* args) { return call_packed(&kllm_attention_prefill_q8_tcgen05, args); }
