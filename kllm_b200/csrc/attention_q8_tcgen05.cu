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
//   warps 8-11       loader: a tile's bytes from the pages into registers a tile ahead, converted to float16 and stored in the
//                    128-byte-swizzled layout that the descriptors name (panels of 64 dims, 8-row groups of 1024 bytes,
//                    the 16-byte piece index XORed with the row index modulo 8).
//   warp 12          issues every tcgen05.mma, one elected thread.
//
// Scales.  Within a tile's step all keys share one exponent eK and one eV: the loader multiplies every key row by
// 2^(ek - eK) and every value row by 2^(ev - eV) as it converts, exactly, as long as the difference is within +-7
// (448 * 2^7 and 2^-9 * 2^-7 are float16 numbers).  It takes the exponents of the tile's first key for eK and eV; keys whose
// pages differ by more wait for a further step over the same tile, in which they are the ones that are seen (page scales of
// one tile are hardly ever so far apart).  So a step has one factor for its scores, one shift for its weights and one
// for the sum, none of them per score.
//
// The output accumulates in TMEM; a row's reference is moved only when its maximum has grown by 2^8 (then the row of the
// accumulator is read, rescaled and written back between two products).  Few row tiles behind a long context are cut
// over the keys: every part leaves its unscaled rows, references and sums, which a second kernel joins in order.
//
// Every wait on an mbarrier is bounded by a cycle count: a wait that runs out raises a flag in shared memory and sets the
// status word, every role leaves its loop, and the CTA frees its TMEM and returns.
#include "q8.cuh"

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
constexpr int THREADS = 512;
constexpr int PANEL = 128 * 128;           // bytes of a panel: 128 rows of 64 float16
constexpr int Q_BYTES = PANELS * PANEL;    // per row tile
constexpr int KV_BYTES = PANELS * PANEL;   // keys or values of a tile
constexpr int STAGES = HD == 64 ? 3 : 2;
constexpr int NOTES = 4;                   // steps described at a time; see note_ring
constexpr int SMEM_BYTES = 1024 + 2 * Q_BYTES + STAGES * 2 * KV_BYTES;
static_assert(SMEM_BYTES <= 226 * 1024, "shared memory");
constexpr unsigned COL_S = 0, COL_O = 256; // scores / weights of the row tiles: 128 columns each; outputs: HD each
constexpr int TMEM_COLS = 512;
constexpr int REGS_SOFTMAX = 168, REGS_LOADER = 120, REGS_ISSUER = 56;
// setmaxnreg moves registers inside the CTA's own allocation (threads x registers at launch)
static_assert(2 * REGS_SOFTMAX + REGS_LOADER + REGS_ISSUER <= THREADS / 128 * (65536 / THREADS), "setmaxnreg budget");
constexpr int PIECES = HD / 16;            // 16-byte pieces of a stored row
constexpr int LOADS = TILE * PIECES / 128; // pieces of the keys (of the values) a loader thread carries
constexpr int E_SPAN = 7;                  // how far a key's exponents may be from its step's

// What the loader says of a step.  note_ring: the note of step t is written once the keys of step t - STAGES have been used,
// for which both softmax groups have passed step t - STAGES - 1; with STAGES <= 3 nobody still reads step t - 4's.
struct Note {
    int key0, ek, ev, last;
    uint32_t member[4];                    // the keys of the tile that this step is for
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
__device__ __forceinline__ void store16(unsigned addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t half2_times(uint32_t x, uint32_t m) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(x), "r"(m));
    return r;
}
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

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
    __shared__ __align__(8) uint64_t bar_q_full[2], bar_s_full[2], bar_p_full[2], bar_o_full[2], bar_note[NOTES];
    __shared__ Note s_note[NOTES];
    __shared__ int s_row[TILE], s_exp[TILE];               // the loader's keys: rows in the stores, exponents (INT_MIN: none)
    __shared__ uint32_t s_left[4];
    __shared__ unsigned s_tmem;
    __shared__ int s_req, s_tok0, s_abort;
    const int split = blockIdx.x % a.splits, kvh = (blockIdx.x / a.splits) % a.n_kv;   // CTAs start in the order of blockIdx.x:
    const int gs = a.n_heads / a.n_kv, tpt = a.tokens_per_tile, per_cta = tpt * a.row_tiles;     // longest key ranges first
    const int warp = warp_index(), lane = threadIdx.x & 31;
    griddep_wait();
    griddep_launch();
    if (threadIdx.x == 0) {
        int tile = (gridDim.x - 1 - blockIdx.x) / (a.n_kv * a.splits), req = -1, tok0 = 0;
        for (int s = 0; s < a.n_requests; s++) {
            const int n = a.q_start[s + 1] - a.q_start[s];
            const int nt = (n + per_cta - 1) / per_cta;
            if (tile < nt) { req = s; tok0 = a.q_start[s] + tile * per_cta; break; }
            tile -= nt;
        }
        if (req >= 0 && min(a.q_start[req + 1], a.n_tokens) <= tok0) req = -1;
        s_req = req; s_tok0 = tok0; s_abort = 0;
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&bar_k_full[i], 128); mbar_init(&bar_k_empty[i], 1);
            mbar_init(&bar_v_full[i], 128); mbar_init(&bar_v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar_q_full[i], ROWS); mbar_init(&bar_s_full[i], 1);
            mbar_init(&bar_p_full[i], ROWS); mbar_init(&bar_o_full[i], 1);
        }
        for (int i = 0; i < NOTES; i++) mbar_init(&bar_note[i], 128);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncthreads();
    const int req = s_req;
    if (req < 0) return;                       // the grid is an upper bound on the tiles
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const int tok0 = s_tok0;
    const int n_tok = min(per_cta, min(a.q_start[req + 1], a.n_tokens) - tok0);       // at least 1
    const int tiles = n_tok > tpt ? 2 : 1;     // row tiles in use
    const int pos0 = a.start_pos[req] + (tok0 - a.q_start[req]);
    const int lo = (a.window > 0 && pos0 + 1 > a.window) ? pos0 + 1 - a.window : 0;
    const int hi = max(pos0 + n_tok, 1);       // one tile at least: every role takes at least one step
    // this part's tiles of keys
    const int first = lo / TILE, all = (hi + TILE - 1) / TILE - first;
    const int per_split = (all + a.splits - 1) / a.splits;
    const int tile_lo = first + min(all, split * per_split), tile_hi = first + min(all, (split + 1) * per_split);
    const bool nothing = tile_lo >= tile_hi;   // a part without keys: its rows' sums are zeros
    volatile int* abort_flag = &s_abort;
    const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;       // swizzled tiles want 1024-byte alignment
    const unsigned sQ = base, sK = base + 2 * Q_BYTES, sV = sK + STAGES * KV_BYTES;

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_ISSUER));
        if (warp == 12 && !nothing) {
            // ---- the issuer: the first scores of both row tiles, then per step and row tile weights x values and the next scores
            constexpr uint32_t IDESC_S = make_idesc_f16(ROWS, TILE, false), IDESC_O = make_idesc_f16(ROWS, HD, true);
            const uint32_t q_lo0 = desc_lo(sQ, 16), k_lo0 = desc_lo(sK, 16), v_lo0 = desc_lo(sV, PANEL);
            auto issue_scores = [&](int x, int stage) {
                const uint32_t q_lo = q_lo0 + (uint32_t)(x * (Q_BYTES >> 4)), k_lo = k_lo0 + (uint32_t)(stage * (KV_BYTES >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t off = (uint32_t)(((kk >> 2) * PANEL + (kk & 3) * 32) >> 4);
                        umma_words(tmem + COL_S + x * TILE, q_lo + off, k_lo + off, IDESC_S, kk > 0);
                    }
                    umma_commit(&bar_s_full[x]);
                    if (x == tiles - 1) umma_commit(&bar_k_empty[stage]);
                }
                __syncwarp();
            };
            bool ok = true;
            for (int x = 0; ok && x < tiles; x++) ok = mbar_wait_warp(&bar_q_full[x], 0, abort_flag, a.status, 2);
            ok = ok && mbar_wait_warp(&bar_k_full[0], 0, abort_flag, a.status, 3);
            if (ok) {
                fence_async_smem();
                tc_fence_after();
                for (int x = 0; x < tiles; x++) issue_scores(x, 0);
            }
            int ks = STAGES == 1 ? 0 : 1, vs = 0;              // stages of the next scores' keys and of these values
            unsigned kp = 0, vp = 0;                           // and their parities
            for (int step = 0; ok; step++) {
                const bool last = s_note[step % NOTES].last != 0;
                ok = mbar_wait_warp(&bar_v_full[vs], vp, abort_flag, a.status, 4);
                for (int x = 0; ok && x < tiles; x++) {
                    // the weights are in tensor memory and the output is rescaled
                    ok = mbar_wait_warp(&bar_p_full[x], (unsigned)step & 1u, abort_flag, a.status, 5);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t v_lo = v_lo0 + (uint32_t)(vs * (KV_BYTES >> 4));
#pragma unroll
                        for (int kk = 0; kk < TILE / 16; kk++)
                            umma_tmem_a_words(tmem + COL_O + x * HD, tmem + COL_S + x * TILE + (unsigned)(kk * 8),
                                              v_lo + (uint32_t)(kk * (2048 >> 4)), IDESC_O, step > 0 || kk > 0);
                        if (x == tiles - 1) umma_commit(&bar_v_empty[vs]);
                        if (last) umma_commit(&bar_o_full[x]);
                    }
                    __syncwarp();
                    if (!last) {
                        if (x == 0) {
                            ok = mbar_wait_warp(&bar_k_full[ks], kp, abort_flag, a.status, 6);
                            if (!ok) break;
                            fence_async_smem();
                            tc_fence_after();
                        }
                        issue_scores(x, ks);           // in issue order behind the product that reads the columns it overwrites
                    }
                }
                if (last) break;
                if (++ks == STAGES) { ks = 0; kp ^= 1u; }
                if (++vs == STAGES) { vs = 0; vp ^= 1u; }
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_LOADER));
        // ---- loader ------------------------------------------------------------------------
        const int tid = threadIdx.x - 256;
        const int* table = a.block_table + (int64_t)req * a.max_blocks;
        int row = -1, exps = INT_MIN;                      // of key tile * 128 + tid
        auto lookup = [&](int tile) {
            row = -1; exps = INT_MIN;
            const int key = tile * TILE + tid;
            if (tile >= tile_hi || key < lo || key >= hi) return;
            const int lp = key / a.page_size;
            if (lp >= a.max_blocks) return;
            const int page = __ldg(table + lp);
            if ((unsigned)page >= (unsigned)a.n_pages) return;
            const int cell = page * a.n_kv + kvh;
            row = cell * a.page_size + key - lp * a.page_size;
            exps = (q8_exponent(__ldg(a.kscale + cell)) << 16) | (q8_exponent(__ldg(a.vscale + cell)) & 0xffff);
        };
        // a thread's pieces: their keys differ by whole groups of 128 / PIECES
        const int piece = tid % PIECES, key_off = tid / PIECES;
        const bool odd_first = PIECES == 8 && piece >= 4;      // the panels of a row at a time on different banks
        uint4 kraw[LOADS], vraw[LOADS];
        auto convert = [&](const uint4 (&raw)[LOADS], unsigned dst, int shift_of, int e_step) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int key = key_off + i * (128 / PIECES);
                const int ee = s_exp[key];
                const bool in = ee != INT_MIN && ((s_left[key >> 5] >> (key & 31)) & 1u);
                const int d = (shift_of ? ee >> 16 : (int)(short)(ee & 0xffff)) - e_step;
                // 2^d as two float16: exponent field d + 15
                const uint32_t m = (uint32_t)((d + 15) << 10) * 0x10001u;
                uint4 x = raw[i];
                if (!in) x = make_uint4(0, 0, 0, 0);
                uint32_t h[8];
                q8_to_f16x4(x.x, h[0], h[1]); q8_to_f16x4(x.y, h[2], h[3]);
                q8_to_f16x4(x.z, h[4], h[5]); q8_to_f16x4(x.w, h[6], h[7]);
                if (in) {
#pragma unroll
                    for (int j = 0; j < 8; j++) h[j] = half2_times(h[j], m);
                }
                const unsigned panel = dst + (unsigned)((piece >> 2) * PANEL);
                const unsigned at0 = panel + swz(key, (piece & 3) * 2), at1 = panel + swz(key, (piece & 3) * 2 + 1);
                if (odd_first) {
                    store16(at1, h[4], h[5], h[6], h[7]);
                    store16(at0, h[0], h[1], h[2], h[3]);
                } else {
                    store16(at0, h[0], h[1], h[2], h[3]);
                    store16(at1, h[4], h[5], h[6], h[7]);
                }
            }
        };
        lookup(tile_lo);
        bool ok = true;
        int stage = 0, step = 0;
        unsigned parity = 1;                                   // of the stages' "empty" barriers: free at first
        for (int tile = tile_lo; ok && tile < tile_hi; tile++) {
            s_row[tid] = row; s_exp[tid] = exps;
            named_sync(1, 128);
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int r = s_row[key_off + i * (128 / PIECES)];
                kraw[i] = vraw[i] = make_uint4(0, 0, 0, 0);
                if (r >= 0) {
                    kraw[i] = __ldg(reinterpret_cast<const uint4*>(a.kcache + (int64_t)r * HD + piece * 16));
                    vraw[i] = __ldg(reinterpret_cast<const uint4*>(a.vcache + (int64_t)r * HD + piece * 16));
                }
            }
            bool left = exps != INT_MIN;                       // this thread's key has not had its step
            const int mine = exps;
            lookup(tile + 1);
            bool done = false;
            while (ok && !done) {
                // the first key that is left names the step's exponents; those near enough join it
                const uint32_t b = __ballot_sync(0xffffffffu, left);
                if (lane == 0) s_left[warp - 8] = b;
                named_sync(1, 128);
                int lead = -1;
#pragma unroll
                for (int w = 3; w >= 0; w--)
                    if (s_left[w]) lead = w * 32 + __ffs(s_left[w]) - 1;
                const int le = lead >= 0 ? s_exp[lead] : 0, ek = le >> 16, ev = (int)(short)(le & 0xffff);
                const bool in = left && abs((mine >> 16) - ek) <= E_SPAN && abs((int)(short)(mine & 0xffff) - ev) <= E_SPAN;
                done = half_all(2, !left || in);               // and everybody has read s_left
                const uint32_t member = __ballot_sync(0xffffffffu, in);
                if (lane == 0) s_left[warp - 8] = member;
                left = left && !in;
                ok = half_all(1, mbar_wait(&bar_k_empty[stage], parity, abort_flag, a.status, 1));
                if (!ok) break;
                Note& note = s_note[step % NOTES];
                if (lane == 0) note.member[warp - 8] = member;
                if (tid == 0) { note.key0 = tile * TILE; note.ek = ek; note.ev = ev; note.last = done && tile + 1 == tile_hi; }
                mbar_arrive(&bar_note[step % NOTES]);
                convert(kraw, sK + stage * KV_BYTES, 1, ek);
                fence_async_smem();
                mbar_arrive(&bar_k_full[stage]);
                ok = half_all(1, mbar_wait(&bar_v_empty[stage], parity, abort_flag, a.status, 7));
                if (!ok) break;
                convert(vraw, sV + stage * KV_BYTES, 0, ev);
                fence_async_smem();
                mbar_arrive(&bar_v_full[stage]);
                if (++stage == STAGES) { stage = 0; parity ^= 1u; }
                step++;
                named_sync(1, 128);                            // s_left and s_row are read
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS_SOFTMAX));
        // ---- softmax: this thread's row is (token, head of the group) of row tile x -----------------------
        const int x = warp >> 2, r = threadIdx.x & 127;
        const int tt = x * tpt + r / gs, hh = r % gs;
        const bool valid = r < tpt * gs && tt < n_tok;
        const int p_row = valid ? pos0 + tt : -1;                           // -1: sees no key
        const int w_row = (a.window > 0) ? p_row + 1 - a.window : 0;
        const int64_t at = (int64_t)(tok0 + tt) * a.n_heads + kvh * gs + hh;
        const unsigned lane_base = (unsigned)((warp & 3) * 32) << 16;
        const unsigned t_s = tmem + lane_base + COL_S + x * TILE, t_o = tmem + lane_base + COL_O + x * HD;
        float m_ref = -INFINITY, l_run = 0.f;
        bool ok = x < tiles && !nothing;
        if (ok) {
            // the row's queries: float16, its power of two in the factor, the scale's sign in the numbers
            const bf16* q = a.q + (int64_t)(tok0 + tt) * a.q_stride + (int64_t)(kvh * gs + hh) * HD;
            uint32_t w[HD / 2];
            int m = 0;
#pragma unroll
            for (int i = 0; i < HD / 8; i++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (valid) {
                    if (a.q_by_eight) {
                        v = *reinterpret_cast<const uint4*>(q + i * 8);
                    } else {
                        const unsigned short* h = reinterpret_cast<const unsigned short*>(q + i * 8);
                        v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
                    }
                }
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
#pragma unroll
                for (int j = 0; j < 4; j++) m = max(m, max((int)(w[4 * i + j] & 0x7fffu) << 16, (int)(w[4 * i + j] & 0x7fff0000u)));
            }
            const bool finite = m < 0x7f800000;
            const float up = finite ? copysignf(q8_pow2(row_shift(m)), a.scale) : 0.f;
            const float factor = finite ? fabsf(a.scale) * kLog2e * q8_pow2(-row_shift(m)) : __int_as_float(0x7fffffff);
            const unsigned dst = sQ + x * Q_BYTES;
#pragma unroll
            for (int i = 0; i < HD / 8; i++) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t two = finite ? w[4 * i + j] : 0u;
                    h[j] = q8_half2(__uint_as_float(two << 16) * up, __uint_as_float(two & 0xffff0000u) * up);
                }
                store16(dst + (unsigned)((i >> 3) * PANEL) + swz(r, i & 7), h[0], h[1], h[2], h[3]);
            }
            fence_async_smem();
            mbar_arrive(&bar_q_full[x]);
            bool last = false;
            for (int step = 0; ok && !last; step++) {
                ok = mbar_wait(&bar_note[step % NOTES], (unsigned)(step / NOTES) & 1u, abort_flag, a.status, 8) &&
                     mbar_wait(&bar_s_full[x], (unsigned)step & 1u, abort_flag, a.status, 9);
                if (!ok) break;
                tc_fence_after();
                const Note& note = s_note[step % NOTES];
                last = note.last != 0;
                // never 0 (a scale of 0, tiny queries): -inf has to stay -inf; NaN stays
                const float product = factor * q8_pow2(note.ek), f = product < 1.1754944e-38f ? 1.1754944e-38f : product;
                const float ev = (float)note.ev;
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
                    for (int j = 0; j < 32; j++) mx4[j & 3] = fmaxf(mx4[j & 3], s[c][j]);
                const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                const float mx = top == -INFINITY ? -INFINITY : fmaf(top, f, ev);
                const bool move = mx > m_ref + kMoveAt;
                float corr = 1.f;
                if (move) {
                    corr = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
                    m_ref = mx;
                }
                const float shift = m_ref == -INFINITY ? ev + kLift : ev - m_ref + kLift;
                float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float pk[32];
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float p0 = fast_exp2(fmaf(s[half * 2 + c][j], f, shift)), p1 = fast_exp2(fmaf(s[half * 2 + c][j + 1], f, shift));
                            sum4[j & 3] += p0;
                            sum4[(j + 1) & 3] += p1;
                            pk[c * 16 + j / 2] = __uint_as_float(q8_half2(p0, p1));
                        }
                    tmem_st32(t_s + half * 32, pk);        // over the first 64 columns of the scores
                }
                l_run = l_run * corr + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])) * q8_pow2(-note.ev);
                if (step > 0 && __any_sync(0xffffffffu, move)) {
                    // rows of this warp rescale what the products so far have added up (rows that did not move multiply by
                    // one); the product of the step before is over, the next one waits for these weights
#pragma unroll
                    for (int cb = 0; cb < HD / 32; cb++) {
                        float t[32];
                        tmem_ld32(t_o + cb * 32, t);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j++) t[j] *= corr;
                        tmem_st32(t_o + cb * 32, t);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar_p_full[x]);
            }
            if (ok) ok = mbar_wait(&bar_o_full[x], 0, abort_flag, a.status, 10);
            if (ok) {
                tc_fence_after();
#pragma unroll
                for (int cb = 0; cb < HD / 32; cb++) {
                    float t[32];
                    tmem_ld32(t_o + cb * 32, t);
                    tmem_ld_wait();
                    if (!valid) continue;
                    if (a.splits == 1) {
                        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint4 pk;
                            pk.x = pack_bf16(t[8 * c] * inv, t[8 * c + 1] * inv);
                            pk.y = pack_bf16(t[8 * c + 2] * inv, t[8 * c + 3] * inv);
                            pk.z = pack_bf16(t[8 * c + 4] * inv, t[8 * c + 5] * inv);
                            pk.w = pack_bf16(t[8 * c + 6] * inv, t[8 * c + 7] * inv);
                            *reinterpret_cast<uint4*>(a.out + at * HD + cb * 32 + 8 * c) = pk;
                        }
                    } else {
                        float* part = a.part_o + (at * a.splits + split) * HD + cb * 32;
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            *reinterpret_cast<float4*>(part + 4 * c) = make_float4(t[4 * c], t[4 * c + 1], t[4 * c + 2], t[4 * c + 3]);
                    }
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
    if (warp == 12)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(TMEM_COLS));
}

}  // namespace

extern "C" int kllm_attention_q8_tcgen05_head_dim() { return HD; }

// Requests' portions: rows q_start[s]..q_start[s+1] of request s start at cache position start_pos[s]; bfloat16 rows.  row_tiles:
// tiles of 128 rows a CTA (1 or 2); splits: parts of the keys, with part_o float32 [n, heads, splits, HD] and part_ml
// float32 [n, heads, splits, 2] where there are several.  status: a device int that a bounded wait which ran out sets (1, 7:
// loader, 2-6: issuer, 8-10: softmax).
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
        kllm_launch((q8_join_kernel<bf16, HD>), dim3((unsigned)(n_tokens * n_heads)), dim3(HD / 4), 0, (cudaStream_t)stream, (bf16*)out,
                    (const float*)part_o, (const float*)part_ml, splits, n_heads, q_start, n_requests);
    }
    KLLM_LAUNCH_STATUS();
}
