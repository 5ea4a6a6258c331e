// A pool of cache pages shared by many sequences: decode attention over it, copies between it and the dense planes of
// prefill, and the eviction of rows that drew little attention.
//
// Pools are [pages][kv_heads][page_rows][head_dim] f16.  Row j of sequence s lies in page table[s][j / page_rows]; a
// row is contiguous, and the rows of one head in one page are.  Every page id is compared with the number of pages
// before it becomes an address: an id that is none reads as zeros, is not written, and sets TM_CUDA_STATUS_BAD_PAGE.
#include "tm_cuda_internal.cuh"
#include "tm_cuda_device.cuh"

namespace {

using tmdev::mma_f16;
using tmdev::smem_addr;

constexpr uint32_t kSeqNone = TM_CUDA_SEQ_NONE;

bool pages_ok(uint32_t head_dim, uint32_t page_rows) {
    return (head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256) &&
           (page_rows == 16 || page_rows == 32 || page_rows == 64 || page_rows == 128 || page_rows == 256);
}
uint32_t log2_of(uint32_t v) {
    uint32_t l = 0;
    while ((1u << l) < v) ++l;
    return l;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {  // zeros where not live
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
// Byte offset of 16-byte chunk `chunk` of row `row` in rows of PITCH bytes: the eight rows that an ldmatrix reads at one
// chunk fall into distinct banks.
template <int PITCH>
__device__ __forceinline__ uint32_t sw(uint32_t row, uint32_t chunk) {
    if (PITCH >= 128) return row * PITCH + ((chunk ^ (row & 7u)) << 4);
    return row * PITCH + ((chunk ^ ((row >> 1) & 3u)) << 4);  // 64-byte rows: two rows per 128 bytes
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// ---- decode attention ------------------------------------------------------------------------------
//
// One new token of every sequence: z_hj = scale q_h . k_j over the rows j in sight, P = softmax(z), out_h = sum_j P_hj v_j,
// and, where a caller counts attention, weights[kv][j] += sum over the group's heads of P_hj.
//
// What bounds it: the cached rows' bytes, 4 head_dim per row and KV head.  So every row is read once for eight query heads
// of its group (with more, a pair for every eight of them, each of which reads the rows again: 32 sequences of up to 4000 rows, one
// KV head of 128, 8 query heads 15 us, 32 heads 28), and the machine's bandwidth is shared out evenly however ragged the lengths are:
// the tiles of 64 rows of all (sequence, KV head) pairs form one line, and CTA i of G takes the i-th of G equal runs of
// it.  Three launches: the vectors (queries and new rows: norm, rotation, f16), the rows, and the join of what the warps
// have found.  The second starts beside the first and waits for it when it has its rows on their way.
//
// What it measured (8 KV heads of 128): the rows of one sequence of 131071 (537 MB) 85 us, 6.3 TB/s, of 32 up to 4095 (343 MB
// with the scores) 61 us, 5.7 TB/s; around them 3 us until the first rows arrive and 3 to 7 us of the join.  (Slices whose
// last eighth went to whichever warp was free measured the same: what ends late waits for the memory, not for work.)
//
// A warp takes 16 rows of each tile through its own ring of cp.async stages and keeps its own running (max, sum, output):
// the warps of a CTA never meet (with the pieces of a pair combined in the CTA, barriers and the next pair's queries took
// 7000 cycles a pair, as long as 250 rows).  The ring runs on across pairs.  Both products are mma.m16n8k16 with the cached
// rows as the 16-row operand and the heads as the 8 columns: S^T = K Q^T, then O^T = V^T P^T, with P transposed in registers.
//
// Accuracy: cached rows are f16, so their products with f16 operands are exact in f32.  Q and P are split into a sum of two
// f16 each (22 bits; Q against a power of two at its largest element, P in units of 2^-14), and every product of a 16-row
// step starts from zero and is added to the f32 sums by a fused multiply-add: results are those of 32-bit arithmetic.  What
// the first f16 leaves is multiplied by 2^12, or it would lie among the subnormals: an element of Q is off by at most 2^-37 of
// the largest where it would be 2^-25, which a large key beside a small element shows, and a weight by at most 2^-51 of the
// largest where it would be 2^-39, which a first row that draws all attention and has a value of zero shows.  (Q's parts have
// sums of their own anyway; for P's apart the rows cost 0.1 us more of 5.4, 22.0 and 8.0, 0.3 of 71.2.)  The second multiply
// hides behind the loads.
constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
constexpr uint32_t kBlock = 16, kTile = kBlock * kAttnWarps;
constexpr float kUnit = 14.0f;  // P and its sums are held times 2^14
constexpr float kLow = 4096.0f;  // the second f16 of an element of Q or P is held times 2^12

template <int HD>
struct attn_cfg {
    static constexpr int PITCH = HD * 2;
    static constexpr uint32_t kPlane = kBlock * PITCH, kStage = 2 * kPlane;  // a warp's 16 keys, then its 16 values
    static constexpr int kStages = HD > 64 ? 3 : 4;
    static constexpr int kCtas = HD == 256 ? 1 : HD == 128 ? 2 : 3;  // an SM
    static constexpr uint32_t kRing = kAttnWarps * kStages * kStage;
    static constexpr uint32_t kQ = HD / 16 * 32 * 16;  // a pair's queries as operands: 16 bytes a lane and 16 dims
    static constexpr bool kQRegs = HD <= 128;          // held in registers, else a copy a warp in shared memory
    static constexpr uint32_t kBytes = kRing + (kQRegs ? 0u : kAttnWarps * kQ);
};
// CTAs of a launch, for which the scratch has room: one to three on each of up to 160 SMs.
constexpr uint32_t most_ctas(uint32_t head_dim) { return 160u * (head_dim == 256 ? 1u : head_dim == 128 ? 2u : 3u); }

struct paged_args {
    const float *q, *k, *v, *q_norm, *k_norm, *inv_freq;
    __half *kp, *vp;
    const uint32_t *table, *pos, *len;
    float *out, *scores;  // scores: only where weights are counted
    uint4 *ops;           // [sequence][pair][16 dims][lane]: the pair's queries as the multiply's operand, high and low halves
    float *factor;        // [sequence][pair][8]: what makes a product of those a score in units of log 2
    // The warps' outputs and (max, sum): of a pair that goes on from another CTA or into one [CTA][0: goes on, 1: begins][8][warp],
    // of a pair that one CTA has whole [sequence][head][warp].
    float *part, *whole;
    float2 *part_ml, *whole_ml;
    const float *w_in;
    float *w_out;
    uint32_t *status;
    uint32_t n_seq, q_stride, kv_stride, heads, kv_heads, group, blocks;  // blocks of up to 8 heads in a group
    uint32_t n_rot, pages, page_log, max_pages, cap, window, ctas;
    float eps, scale_log2e;
};

__device__ __forceinline__ uint32_t first_row(uint32_t len, uint32_t window) {
    return window != 0u && len >= window ? len + 1u - window : 0u;
}
// Tiles of one (sequence, KV head) pair; none for a sequence that takes no part or is full.
__device__ __forceinline__ uint32_t pair_tiles(uint32_t len, const paged_args &a) {
    return len >= a.cap ? 0u : len / kTile - first_row(len, a.window) / kTile + 1u;
}
// The line of all pairs' tiles and the CTAs that share it, each with one tile at least, so that the pieces of a pair lie in
// consecutive CTAs: CTA i has `each` tiles, or one more if i < extra.  (Entry point: T < 2^32.)
struct line {
    uint32_t ctas, each, extra;
    __device__ __forceinline__ line(uint32_t T, const paged_args &a) {
        ctas = min(T, a.ctas);
        each = ctas != 0u ? T / ctas : 0u;
        extra = T - each * ctas;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + min(i, extra); }
    __device__ __forceinline__ uint32_t owner(uint32_t t) const {
        const uint32_t longer = extra * (each + 1u);
        return t < longer ? t / (each + 1u) : extra + (t - longer) / each;
    }
};
// The sequences' lengths.  The second and third launch read them (and pages, cached rows, earlier weights) before their waits:
// all that has been complete since before the first let them start.  Until the wait it is read from L2, past whatever an SM
// has kept; the first 32 stay in the lanes of each warp.
struct lengths {
    uint32_t held;
    __device__ __forceinline__ lengths(const paged_args &a) {
        const uint32_t lane = threadIdx.x & 31u;
        held = lane < a.n_seq ? __ldcg(a.len + lane) : kSeqNone;
    }
    __device__ __forceinline__ uint32_t lane_of(const paged_args &a, uint32_t s0) const {  // of sequence s0 + lane
        const uint32_t s = s0 + (threadIdx.x & 31u);
        return s0 == 0u ? held : s < a.n_seq ? __ldcg(a.len + s) : kSeqNone;
    }
    __device__ __forceinline__ uint32_t of(const paged_args &a, uint32_t s) const {  // the same sequence for all lanes
        return s < 32u ? __shfl_sync(0xffffffffu, held, s) : __ldcg(a.len + s);
    }
};
// Tiles of one head's pairs of the sequences below `upto` (whole warps call it).
__device__ __forceinline__ uint32_t tiles_before(const lengths &lens, uint32_t upto, const paged_args &a) {
    uint32_t n = 0;
    for (uint32_t s0 = 0; s0 < upto; s0 += 32u) {
        const uint32_t tiles = pair_tiles(lens.lane_of(a, s0), a);
        n += s0 + (threadIdx.x & 31u) < upto ? tiles : 0u;
    }
    return __reduce_add_sync(0xffffffffu, n);
}

// A tile of the line.
struct cursor {
    uint32_t s, pair, t, nt, len, start;
    __device__ __forceinline__ void enter(const paged_args &a, uint32_t rows) {
        len = rows;
        nt = pair_tiles(len, a);
        start = first_row(len, a.window);
    }
    // To the next pair; behind the last one of all it stays at a sequence that is none.
    __device__ __forceinline__ void next_pair(const lengths &lens, const paged_args &a) {
        t = 0;
        if (++pair < a.kv_heads * a.blocks) return;
        pair = 0;
        for (++s; s < a.n_seq; ++s) {
            enter(a, lens.of(a, s));
            if (nt != 0u) break;
        }
    }
};

// The vectors: a warp norms and rotates one query head, or a KV head's new key, and stores it.  Its latency is hidden by
// nothing, so everything it needs is asked for at once.
//
// y / rms(y) * w, then the pairs (i, i + half) turned, in T; `row` is the warp's.
__device__ __forceinline__ float inverse_rms(float mean, float eps) { return 1.0f / sqrtf(mean + eps); }
__device__ __forceinline__ double inverse_rms(double mean, float eps) { return rsqrt(mean + (double)eps); }
__device__ __forceinline__ void sine_cosine(float x, float &s, float &c) { sincosf(x, &s, &c); }
__device__ __forceinline__ void sine_cosine(float x, double &s, double &c) { sincos((double)x, &s, &c); }
template <int HD, typename T, int EPL, int PAIRS>
__device__ __forceinline__ void norm_and_turn(T *row, const float (&y)[EPL], const float (&w)[EPL], const float (&freq)[PAIRS], float pos,
                                              uint32_t half, float eps) {
    const uint32_t lane = threadIdx.x & 31u;
    T ss = 0;
#pragma unroll
    for (int r = 0; r < EPL; ++r) ss += (T)y[r] * (T)y[r];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T inv = inverse_rms(ss / (T)HD, eps);
#pragma unroll
    for (int r = 0; r < EPL; ++r) row[lane + 32 * r] = (T)y[r] * inv * (T)w[r];
    __syncwarp();
#pragma unroll
    for (int r = 0; r < PAIRS; ++r) {
        const uint32_t i = lane + 32 * r;
        if (i < half) {
            T sn, c;
            sine_cosine(pos * freq[r], sn, c);
            const T x0 = row[i], x1 = row[i + half];
            row[i] = x0 * c - x1 * sn;
            row[i + half] = x0 * sn + x1 * c;
        }
    }
    __syncwarp();
}

template <int HD>
__global__ void __launch_bounds__(256) attention_paged_vectors_kernel(const paged_args a) {
    constexpr int EPL = HD / 32;
    __shared__ double rows[8][HD];
    tmdev::pdl_wait();
    tmdev::pdl_trigger();  // the next kernel may read what those before this one have written
    const uint32_t warp = tmdev::warp_index(), lane = threadIdx.x & 31u, per = a.heads + a.kv_heads;
    const uint64_t at = (uint64_t)blockIdx.x * 8u + warp;
    const uint32_t s = (uint32_t)(at / per), x = (uint32_t)(at % per);
    if (s >= a.n_seq) return;
    const bool is_k = x >= a.heads;
    const uint32_t kvh = x - a.heads, len = a.len[s], pos = a.pos[s];
    const float *src = is_k ? a.k + (size_t)s * a.kv_stride + (size_t)kvh * HD : a.q + (size_t)s * a.q_stride + (size_t)x * HD;
    const float *nw = is_k ? a.k_norm : a.q_norm, *vs = a.v + (size_t)s * a.kv_stride + (size_t)kvh * HD;
    const uint32_t half = a.n_rot / 2u;
    constexpr int kPairs = HD > 64 ? HD / 64 : 1;  // rotation pairs of a lane, at most
    float y[EPL], w[EPL], v[EPL], freq[kPairs];
#pragma unroll
    for (int r = 0; r < EPL; ++r) {
        y[r] = src[lane + 32 * r];
        w[r] = nw[lane + 32 * r];
        v[r] = is_k ? vs[lane + 32 * r] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kPairs; ++r) freq[r] = lane + 32 * r < half ? a.inv_freq[lane + 32 * r] : 0.0f;
    const uint32_t id = is_k && len < a.cap ? a.table[(size_t)s * a.max_pages + (len >> a.page_log)] : 0u;
    if (len >= a.cap) {
        if (x == 0u && lane == 0 && len != kSeqNone) atomicOr(a.status, TM_CUDA_STATUS_PAST_CAPACITY);
        return;
    }
    if (is_k) {
        if (id >= a.pages) {
            if (lane == 0) atomicOr(a.status, TM_CUDA_STATUS_BAD_PAGE);
            return;
        }
        // The stored key is what every later token meets: worked out in 64 bits, so that what is rounded to f16 is right in every bit
        // of f32.  (In 32 bits one element in some thousands comes to lie on the other side of a tie of f16, and a whole step of it
        // away.  The queries' warps take as long, so this costs nothing.)
        double *row = rows[warp];
        norm_and_turn<HD>(row, y, w, freq, (float)pos, half, a.eps);
        const size_t to = ((((size_t)id * a.kv_heads + kvh) << a.page_log) + (len & ((1u << a.page_log) - 1u))) * HD;
#pragma unroll
        for (int r = 0; r < EPL; ++r) {
            a.kp[to + lane + 32 * r] = __float2half_rn((float)row[lane + 32 * r]);
            a.vp[to + lane + 32 * r] = __float2half_rn(v[r]);
        }
        return;
    }
    float *row = (float *)rows[warp];
    norm_and_turn<HD>(row, y, w, freq, (float)pos, half, a.eps);
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < EPL; ++r) top = fmaxf(top, fabsf(row[lane + 32 * r]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // q = 2^e (hi + lo / kLow), |hi| < 2; a vector of zeros, infinities or NaN keeps e = 0
    int e = (int)((__float_as_uint(top) >> 23) & 0xffu) - 127;
    e = top > 0.0f && top < INFINITY ? max(-120, min(120, e)) : 0;
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    const uint32_t in_group = x % a.group, h = in_group % 8u;
    const size_t pair = (size_t)s * a.kv_heads * a.blocks + x / a.group * a.blocks + in_group / 8u;
    if (lane == 0) a.factor[pair * 8 + h] = a.scale_log2e * __uint_as_float((uint32_t)(127 + e) << 23);
    for (uint32_t i = lane; i < HD / 4; i += 32u) {  // lane 4 h + t of the operand for 16 dims: dims 2t, 2t + 1, 2t + 8, 2t + 9
        const float *d = row + i / 4u * 16u + i % 4u * 2u;
        const float z0 = d[0] * down, z1 = d[1] * down, z2 = d[8] * down, z3 = d[9] * down;
        const __half2 h0 = __floats2half2_rn(z0, z1), h1 = __floats2half2_rn(z2, z3);
        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
        a.ops[(pair * (HD / 16) + i / 4u) * 32 + h * 4u + i % 4u] =
            make_uint4(bits(h0), bits(h1), bits(__floats2half2_rn((z0 - f0.x) * kLow, (z1 - f0.y) * kLow)),
                       bits(__floats2half2_rn((z2 - f1.x) * kLow, (z3 - f1.y) * kLow)));
    }
}

template <int HD>
__global__ void __launch_bounds__(kAttnThreads, attn_cfg<HD>::kCtas) attention_paged_kernel(const paged_args a) {
    using C = attn_cfg<HD>;
    constexpr int PITCH = C::PITCH, STAGES = C::kStages, KT = HD / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    const uint32_t warp = tmdev::warp_index(), lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t ring = smem_addr(smem) + warp * (STAGES * C::kStage);
    uint4 *const q_copy = (uint4 *)(smem + C::kRing + (C::kQRegs ? 0u : warp * C::kQ));
    tmdev::pdl_trigger();

    // ---- this CTA's run of tiles ----
    const uint32_t pairs = a.kv_heads * a.blocks;
    const lengths lens(a);
    const line all(tiles_before(lens, a.n_seq, a) * pairs, a);
    if (blockIdx.x >= all.ctas) {
        tmdev::pdl_wait();
        return;
    }
    const uint32_t u0 = all.begin(blockIdx.x);
    uint32_t left = all.begin(blockIdx.x + 1u) - u0;
    cursor at;
    {
        uint32_t before = 0;  // tiles of the sequences before the one that tile u0 belongs to
        at.s = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32u) {
            const uint32_t n = pair_tiles(lens.lane_of(a, s0), a) * pairs;
            uint32_t incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= (uint32_t)o) incl += up;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + incl > u0);
            if (past) {
                const int first = __ffs(past) - 1;
                at.s = s0 + first;
                before += __shfl_sync(0xffffffffu, incl - n, first);
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        at.enter(a, lens.of(a, at.s));
        at.pair = (u0 - before) / at.nt;
        at.t = (u0 - before) % at.nt;
    }

    // ---- the ring of cached rows: `ahead` is the tile whose page was asked for last, `coming` tiles are not on their way ----
    const uint32_t page_low = (1u << a.page_log) - 1u;
    cursor ahead = at;
    uint32_t coming = left, ahead_id = 0u, fill = 0u;
    bool waited = false;
    auto wait = [&] {  // for the vectors
        if (!waited) tmdev::pdl_wait();
        waited = true;
    };
    auto block_of = [&](const cursor &c) { return (c.start / kTile + c.t) * kAttnWarps + warp; };
    auto in_sight = [](const cursor &c, uint32_t blk) { return blk * kBlock <= c.len && blk * kBlock + (kBlock - 1u) >= c.start; };
    auto ask = [&](bool first) {
        const uint32_t blk = block_of(ahead), *page = a.table + (size_t)ahead.s * a.max_pages + (blk * kBlock >> a.page_log);
        ahead_id = !in_sight(ahead, blk) ? 0u : first ? __ldcg(page) : *page;
    };
    auto load = [&](bool first) {
        if (coming != 0u) {
            const uint32_t blk = block_of(ahead);
            if (in_sight(ahead, blk)) {
                if (first && ahead.len - blk * kBlock < kBlock) wait();  // the new row is among these
                const bool page = ahead_id < a.pages;
                if (!page && lane == 0) atomicOr(a.status, TM_CUDA_STATUS_BAD_PAGE);
                const uint32_t kvh = ahead.pair / a.blocks;
                const size_t row0 = (((size_t)(page ? ahead_id : 0u) * a.kv_heads + kvh) << a.page_log) + (blk * kBlock & page_low);
                const uint32_t dst = ring + fill * C::kStage;
#pragma unroll
                for (int c = 0; c < KT; ++c) {
                    const uint32_t e = c * 32 + lane, r = e / (HD / 8), ch = e % (HD / 8), j = blk * kBlock + r;
                    const bool live = page && j >= ahead.start && j <= ahead.len;  // the rest is zeros
                    cp_async16(dst + sw<PITCH>(r, ch), a.kp + (row0 + r) * HD + ch * 8u, live);
                    cp_async16(dst + C::kPlane + sw<PITCH>(r, ch), a.vp + (row0 + r) * HD + ch * 8u, live);
                }
            }
            if (--coming != 0u) {
                if (++ahead.t >= ahead.nt) ahead.next_pair(lens, a);
                ask(first);
            }
        }
        fill = fill + 1u == STAGES ? 0u : fill + 1u;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask(true);
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) load(true);
    wait();

    uint32_t stage = 0u;
#pragma unroll 1
    while (left != 0u) {
        // ---- a run of one pair's tiles ----
        const uint32_t s = at.s, len = at.len, start = at.start, tn = min(at.nt - at.t, left);
        const uint32_t kvh = at.pair / a.blocks, hb = at.pair % a.blocks;
        const uint32_t head0 = kvh * a.group + hb * 8u, heads = min(8u, a.group - hb * 8u);
        const bool begins = at.t == 0u, ends = at.t + tn == at.nt;
        const size_t pair = (size_t)s * pairs + at.pair;
        // (columns of no head hold what the scratch holds: a column of the products depends on nothing but its own)
        uint4 qr[C::kQRegs ? KT : 1];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const uint4 v = a.ops[(pair * KT + kt) * 32 + lane];
            if (C::kQRegs) qr[C::kQRegs ? kt : 0] = v;
            else q_copy[kt * 32 + lane] = v;  // (each lane reads back its own)
        }
        const float f0 = a.factor[pair * 8 + 2 * t], f1 = a.factor[pair * 8 + 2 * t + 1];
        float o[KT][4];
#pragma unroll
        for (int i = 0; i < KT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;  // heads 2t and 2t + 1; l: this lane's rows
        float *scores = a.scores ? a.scores + ((size_t)s * a.kv_heads + kvh) * a.cap * a.group + hb * 8u + 2 * t : nullptr;

#pragma unroll 1
        for (uint32_t i = 0; i < tn; ++i) {
            const uint32_t j0 = ((start / kTile + at.t + i) * kAttnWarps + warp) * kBlock;
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();  // this block has landed for all lanes, and all have read the one before it
            load(false);
            const uint32_t kb = ring + stage * C::kStage, vb = kb + C::kPlane;
            stage = stage + 1u == STAGES ? 0u : stage + 1u;
            if (j0 > len || j0 + (kBlock - 1u) < start) continue;
            float hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                uint32_t a0, a1, a2, a3;
                ldsm_x4(kb + sw<PITCH>(lane & 15u, kt * 2 + (lane >> 4)), a0, a1, a2, a3);
                const uint4 b = C::kQRegs ? qr[C::kQRegs ? kt : 0] : q_copy[kt * 32 + lane];
                mma_f16(hi, a0, a1, a2, a3, b.x, b.y);
                mma_f16(lo, a0, a1, a2, a3, b.z, b.w);
            }
            // rows j0 + g and j0 + g + 8, heads 2t and 2t + 1
            const uint32_t ja = j0 + g, jb = ja + 8u;
            const bool see_a = ja >= start && ja <= len, see_b = jb >= start && jb <= len;
            // (z - z: an infinity is a NaN from here on.  Only an infinite key makes one, and with which sign would hang on how the
            // query was split.)
            auto score = [](float z, float f) { return fmaf(z, f, z - z); };
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = fmaf(lo[i], 1.0f / kLow, hi[i]);
            const float s0 = see_a ? score(z[0], f0) : -INFINITY, s1 = see_a ? score(z[1], f1) : -INFINITY;
            const float s2 = see_b ? score(z[2], f0) : -INFINITY, s3 = see_b ? score(z[3], f1) : -INFINITY;
            if (scores) {
                float *row = scores + (size_t)ja * a.group;
                if (see_a && 2 * t < heads) row[0] = s0;
                if (see_a && 2 * t + 1 < heads) row[1] = s1;
                row += (size_t)8 * a.group;
                if (see_b && 2 * t < heads) row[0] = s2;
                if (see_b && 2 * t + 1 < heads) row[1] = s3;
            }
            float x0 = fmaxf(s0, s2), x1 = fmaxf(s1, s3);
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, sh));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, sh));
            }
            x0 = fmaxf(x0, m0);
            x1 = fmaxf(x1, m1);
            const float d0 = x0 == -INFINITY ? 0.0f : x0, d1 = x1 == -INFINITY ? 0.0f : x1;
            const float al0 = exp2f(m0 - d0), al1 = exp2f(m1 - d1);
            m0 = x0;
            m1 = x1;
            const float p0 = exp2f(s0 - d0 + kUnit), p1 = exp2f(s1 - d1 + kUnit);
            const float p2 = exp2f(s2 - d0 + kUnit), p3 = exp2f(s3 - d1 + kUnit);
            l0 = fmaf(l0, al0, p0 + p2);
            l1 = fmaf(l1, al1, p1 + p3);
            const __half2 pa = __floats2half2_rn(p0, p1), pb = __floats2half2_rn(p2, p3);
            const float2 fa = __half22float2(pa), fb = __half22float2(pb);
            const uint32_t h0 = transpose8x8(bits(pa)), h1 = transpose8x8(bits(pb));
            const uint32_t r0 = transpose8x8(bits(__floats2half2_rn((p0 - fa.x) * kLow, (p1 - fa.y) * kLow)));
            const uint32_t r1 = transpose8x8(bits(__floats2half2_rn((p2 - fb.x) * kLow, (p3 - fb.y) * kLow)));
            const uint32_t mat = lane >> 3, vr = (lane & 7u) + (mat >> 1) * 8u;
#pragma unroll
            for (int mt = 0; mt < KT; ++mt) {
                uint32_t a0, a1, a2, a3;
                ldsm_x4_t(vb + sw<PITCH>(vr, mt * 2 + (mat & 1u)), a0, a1, a2, a3);
                float d[4] = {0, 0, 0, 0}, e[4] = {0, 0, 0, 0};
                mma_f16(d, a0, a1, a2, a3, h0, h1);
                mma_f16(e, a0, a1, a2, a3, r0, r1);
                o[mt][0] = fmaf(o[mt][0], al0, fmaf(e[0], 1.0f / kLow, d[0]));
                o[mt][1] = fmaf(o[mt][1], al1, fmaf(e[1], 1.0f / kLow, d[1]));
                o[mt][2] = fmaf(o[mt][2], al0, fmaf(e[2], 1.0f / kLow, d[2]));
                o[mt][3] = fmaf(o[mt][3], al1, fmaf(e[3], 1.0f / kLow, d[3]));
            }
        }
        // ---- what this warp has found (zeros, where it saw no row) ----
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
            l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
        }
        const bool whole = begins && ends;
        const size_t piece = whole ? ((size_t)s * a.heads + head0) * kAttnWarps + warp
                                   : ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * 8 * kAttnWarps + warp;  // of head 0; then every 4th
        float *to = whole ? a.whole : a.part;
        float2 *ml = whole ? a.whole_ml : a.part_ml;
#pragma unroll
        for (uint32_t e = 0; e < 2u; ++e) {
            const uint32_t h = 2 * t + e;
            if (h >= heads) continue;
            if (g == 0) ml[piece + h * kAttnWarps] = e ? make_float2(m1, l1) : make_float2(m0, l0);
            float *row = to + (piece + h * kAttnWarps) * HD + g;
#pragma unroll
            for (int mt = 0; mt < KT; ++mt) {
                row[mt * 16] = o[mt][e];
                row[mt * 16 + 8] = o[mt][2 + e];
            }
        }
        left -= tn;
        if (left != 0u) at.next_pair(lens, a);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Joins the warps' pieces of every pair (a CTA takes DIMS of a head, a warp a piece), and counts the attention of stretches
// of rows (the CTAs behind those).  What needs neither pieces nor scores is done while the rows are still being read, and
// every warp finds the maximum of all pieces for itself, so that nothing waits for it but the last sums.  (Counting CTAs are as many
// as rows that the tables have room for; those behind a sequence's last row look at its length and leave: 64 sequences of up to 1000
// rows, 8 KV heads, tables for 1000 rows 41.5 us, for 16384 62.7, for 131072 205.)
constexpr uint32_t kCountEach = 4;
template <int HD, int DIMS, uint32_t kJoinWarps, int kBatch>  // kBatch: pieces of a warp on their way at a time
__global__ void __launch_bounds__(32 * kJoinWarps) attention_paged_join_kernel(const paged_args a) {
    constexpr int EPL = DIMS / 32;
    constexpr uint32_t kParts = HD / DIMS, kJoinThreads = 32 * kJoinWarps, kCountRows = kCountEach * kJoinThreads;
    __shared__ float sm[32], sl[32], so[kJoinWarps][DIMS];
    tmdev::pdl_trigger();
    const uint32_t s = blockIdx.y, tid = threadIdx.x, warp = tmdev::warp_index(), lane = tid & 31u;
    const lengths lens(a);
    const uint32_t len = lens.of(a, s), nt = pair_tiles(len, a), joining = a.heads * kParts;
    const bool joins = blockIdx.x < joining;
    const uint32_t head = blockIdx.x / kParts, d0 = blockIdx.x % kParts * DIMS;  // (of one that joins)
    const uint32_t kvh = joins ? head / a.group : (blockIdx.x - joining) % a.kv_heads;
    const uint32_t row0 = joins ? 0u : (blockIdx.x - joining) / a.kv_heads * kCountRows, start = first_row(len, a.window);
    if (nt == 0u || row0 > len) {
        tmdev::pdl_wait();
        return;
    }
    const size_t base = ((size_t)s * a.kv_heads + kvh) * a.cap;
    float w[kCountEach];
    __align__(16) float z[kCountEach][4];
    if (!joins) {
#pragma unroll
        for (uint32_t r = 0; r < kCountEach; ++r) {
            const uint32_t j = row0 + r * kJoinThreads + tid;
            w[r] = a.w_in && j < len ? __ldcg(a.w_in + base + j) : 0.0f;  // the new row has drawn nothing before
        }
    }
    const uint32_t pairs = a.kv_heads * a.blocks;
    const line all(tiles_before(lens, a.n_seq, a) * pairs, a);
    const uint32_t before = tiles_before(lens, s, a) * pairs;
    // The pieces of a head: `n` of them, 4 a CTA; CTA i0 has begun the pair, the others carry on.
    struct pieces {
        uint32_t n;
        bool whole;
        size_t base;
        __device__ __forceinline__ size_t operator[](uint32_t i) const {  // (the first CTA's lie a block of 8 heads further on)
            const uint32_t cta = i / kAttnWarps;
            return base + (whole || cta == 0u ? 0u : (cta * 2u - 1u) * 8u * kAttnWarps) + i % kAttnWarps;
        }
    };
    auto of = [&](uint32_t head) {
        const uint32_t in_group = head % a.group, u = before + (kvh * a.blocks + in_group / 8u) * nt, i0 = all.owner(u);
        pieces p;
        p.n = (all.owner(u + nt - 1u) - i0 + 1u) * kAttnWarps;
        p.whole = p.n == (uint32_t)kAttnWarps;
        p.base = p.whole ? ((size_t)s * a.heads + head) * kAttnWarps : ((size_t)i0 * 2 + 1) * 8 * kAttnWarps + in_group % 8u * kAttnWarps;
        return p;
    };
    if (joins) {
        const pieces p = of(head);
        tmdev::pdl_wait();
        const float *rows = p.whole ? a.whole : a.part;
        const float2 *mls = p.whole ? a.whole_ml : a.part_ml;
        float top = -INFINITY, L = 0.0f, O[EPL];
#pragma unroll
        for (int r = 0; r < EPL; ++r) O[r] = 0.0f;
        float2 ml[kBatch];
        float ob[kBatch][EPL];
        auto fetch = [&](uint32_t i) {
#pragma unroll
            for (int c = 0; c < kBatch; ++c) {
                const bool live = i + c * kJoinWarps < p.n;
                const size_t x = p[live ? i + c * kJoinWarps : 0u];
                ml[c] = live ? mls[x] : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int r = 0; r < EPL; ++r) ob[c][r] = live ? rows[x * HD + d0 + lane + 32 * r] : 0.0f;
            }
        };
        fetch(warp);
#pragma unroll 4
        for (uint32_t i = lane; i < p.n; i += 32u) top = fmaxf(top, mls[p[i]].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float use = top == -INFINITY ? 0.0f : top;
        for (uint32_t i = warp; i < p.n;) {
#pragma unroll
            for (int c = 0; c < kBatch; ++c) {
                const float f = exp2f(ml[c].x - use);  // a warp that saw no row: 0
                L = fmaf(f, ml[c].y, L);
#pragma unroll
                for (int r = 0; r < EPL; ++r) O[r] = fmaf(f, ob[c][r], O[r]);
            }
            i += kBatch * kJoinWarps;
            if (i < p.n) fetch(i);
        }
        if (lane == 0) sl[warp] = L;
#pragma unroll
        for (int r = 0; r < EPL; ++r) so[warp][lane + 32 * r] = O[r];
        __syncthreads();
        for (uint32_t d = tid; d < (uint32_t)DIMS; d += kJoinThreads) {
            float l = 0.0f, o = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < kJoinWarps; ++x) {
                l += sl[x];
                o += so[x][d];
            }
            a.out[((size_t)s * a.heads + head) * HD + d0 + d] = o / l + (o - o);  // (NaN of an infinite value, as of a key)
        }
        return;
    }
    tmdev::pdl_wait();
#pragma unroll
    for (uint32_t r = 0; r < kCountEach; ++r) {
        const uint32_t j = row0 + r * kJoinThreads + tid;
        const bool seen = j >= start && j <= len;
        const float *row = a.scores + (base + j) * a.group;
        if (a.group % 4u == 0u) {
            if (seen) *(float4 *)z[r] = *(const float4 *)row;
        } else {
#pragma unroll
            for (uint32_t h = 0; h < 4u; ++h) z[r][h] = seen && h < a.group ? row[h] : 0.0f;
        }
    }
    for (uint32_t x = warp; x < a.group; x += kJoinWarps) {  // a head's maximum and sum, a lane a piece
        const pieces p = of(kvh * a.group + x);
        const float2 *mls = p.whole ? a.whole_ml : a.part_ml;
        float M = -INFINITY, L = 0.0f;
        for (uint32_t i = lane; i < p.n; i += 32u) {
            const float2 ml = mls[p[i]];
            const float top = fmaxf(M, ml.x), use = top == -INFINITY ? 0.0f : top;
            L = fmaf(L, exp2f(M - use), exp2f(ml.x - use) * ml.y);
            M = top;
        }
        float top = M;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        L *= exp2f(M - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane == 0) {
            sm[x] = top - kUnit;
            sl[x] = 1.0f / L;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kCountEach; ++r) {
        const uint32_t j = row0 + r * kJoinThreads + tid;
        if (j > len) break;
        if (j >= start) {
            float sum = 0.0f;
#pragma unroll
            for (uint32_t h = 0; h < 4u; ++h)
                if (h < a.group) sum = fmaf(exp2f(z[r][h] - sm[h]), sl[h], sum);
            for (uint32_t h = 4; h < a.group; ++h) sum = fmaf(exp2f(a.scores[(base + j) * a.group + h] - sm[h]), sl[h], sum);
            w[r] += sum;
        }
        a.w_out[base + j] = w[r];
    }
}

// Where the parts of the scratch lie, in bytes; `end` is its size.
struct scratch_parts {
    size_t ops, factor, part, part_ml, whole, whole_ml, scores, end;
    scratch_parts(uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint64_t cap, bool weights) {
        const size_t pairs = (size_t)n_seq * kv_heads * ((heads / kv_heads + 7u) / 8u), rows = (size_t)n_seq * heads * kAttnWarps;
        const size_t pieces = (size_t)most_ctas(head_dim) * 2 * 8 * kAttnWarps;
        ops = 0;
        factor = ops + pairs * (head_dim / 16) * 32 * 16;
        part = factor + pairs * 32;
        part_ml = part + pieces * head_dim * 4;
        whole = part_ml + pieces * 8;
        whole_ml = whole + rows * head_dim * 4;
        scores = whole_ml + rows * 8;
        end = scores + (weights ? (size_t)n_seq * heads * cap * 4 : 0);
    }
};

template <int HD>
cudaError_t launch_paged(tm_cuda_ctx *ctx, paged_args a) {
    using C = attn_cfg<HD>;
    static std::atomic<bool> attr_done[64] = {};  // per device; contexts of a process share it
    const int device = ctx->device;
    if (device < 0 || device >= 64 || !attr_done[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(attention_paged_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kBytes);
        if (e != cudaSuccess) return e;
        if (device >= 0 && device < 64) attr_done[device].store(true, std::memory_order_release);
    }
    // At most: tiles of a pair, pairs, and with these the CTAs.
    const uint32_t whole = (a.cap + kTile - 1) / kTile, seen = a.window && a.window < a.cap ? (a.window + kTile - 2) / kTile + 1u : whole;
    const uint32_t tiles = seen < whole ? seen : whole, pairs = a.n_seq * a.kv_heads * a.blocks;
    const uint32_t most = min((uint32_t)(C::kCtas * ctx->sm_count), most_ctas(HD));
    a.ctas = (uint32_t)min((uint64_t)tiles * pairs, (uint64_t)most);
    const uint64_t vectors = (uint64_t)a.n_seq * (a.heads + a.kv_heads);
    cudaError_t e = tm_launch_pdl(ctx, attention_paged_vectors_kernel<HD>, dim3((uint32_t)((vectors + 7) / 8)), dim3(256), 0, a);
    if (e == cudaSuccess) e = tm_launch_pdl(ctx, attention_paged_kernel<HD>, dim3(a.ctas), dim3(kAttnThreads), C::kBytes, a);
    if (e != cudaSuccess) return e;
    // The join.  Heads that find a place at once: a CTA of eight warps each (20 sequences of 300 rows, 8 heads of 256: 8.3 us, with
    // four warps 8.4; 4 of 500, 40 heads of 128: 7.1, 8.6), else four (60 of 1000, 10 heads of 64: 11.8, with eight 14.0).  A pair
    // in many pieces: its dims are cut into CTAs of 32, if all of these find a place (one of 30000 rows, 8 heads of 256: 20, not
    // cut 44; of 131071, 32 heads of 128: 92, 95; 4 of 2000, 16 heads: 10.6, but 10.3), whose warps read twenty pieces at once, or
    // ten, which takes fewer registers, where the CTAs that count weights are more than find a place beside them (131071: 111, 106).
    const uint32_t pieces = kAttnWarps * min(tiles, a.ctas / pairs + 2u), places = 2u * (uint32_t)ctx->sm_count;
    const uint64_t heads = (uint64_t)a.heads * a.n_seq;
    const bool cut = pieces > 64u && heads * (HD / 32) <= places, wide = cut || heads <= 2u * places;
    const uint32_t rows = kCountEach * 32u * (wide ? 8u : 4u), count = a.w_out ? a.kv_heads * ((a.cap + rows - 1) / rows) : 0u;
    const dim3 grid(a.heads * (cut ? HD / 32 : 1) + count, a.n_seq);
    return cut && (uint64_t)grid.x * a.n_seq <= places
               ? tm_launch_pdl(ctx, attention_paged_join_kernel<HD, 32, 8, 20>, grid, dim3(256), 0, a)
           : cut  ? tm_launch_pdl(ctx, attention_paged_join_kernel<HD, 32, 8, 10>, grid, dim3(256), 0, a)
           : wide ? tm_launch_pdl(ctx, attention_paged_join_kernel<HD, HD, 8, 3>, grid, dim3(256), 0, a)
                  : tm_launch_pdl(ctx, attention_paged_join_kernel<HD, HD, 4, 2>, grid, dim3(128), 0, a);
}

// ---- copies between dense planes and pages ---------------------------------------------------------
//
// Moves 4 head_dim bytes a row and KV head each way and computes nothing: 16 bytes a thread and load, all loads of a
// thread before its first store.  A CTA takes up to 64 rows of one run, one head, keys or values.  Bound by the memory:
// 670 MB (32 sequences of up to 4096 rows, 8 heads of 128) 89 us, 7.5 TB/s of reads and writes together, of which a part is the
// 126 MB of L2's (a plain copy of 4 GB: 6.5 TB/s).
constexpr uint32_t kCopyRows = 64, kCopyThreads = 256;
struct copy_runs {
    uint32_t n;
    uint32_t tile0[TM_CUDA_PREFILL_SEGMENTS + 1];
    uint32_t seq[TM_CUDA_PREFILL_SEGMENTS], at[TM_CUDA_PREFILL_SEGMENTS], row0[TM_CUDA_PREFILL_SEGMENTS], rows[TM_CUDA_PREFILL_SEGMENTS];
};
struct copy_args {
    __half *kc, *vc, *kp, *vp;
    const uint32_t *table;
    uint32_t *status;
    uint32_t pages, page_log, max_pages, kv_heads, cap;
};

template <int HD, bool TO_PAGES>
__global__ void __launch_bounds__(kCopyThreads) kv_pages_copy_kernel(const copy_args a, const __grid_constant__ copy_runs runs) {
    constexpr uint32_t kChunks = HD / 8, kEach = kCopyRows * kChunks / kCopyThreads;  // 16-byte chunks of a row; a thread's
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    uint32_t r = 0;
    while (r + 1u < runs.n && runs.tile0[r + 1u] <= blockIdx.x) ++r;
    const uint32_t first = (blockIdx.x - runs.tile0[r]) * kCopyRows, rows = min(kCopyRows, runs.rows[r] - first);
    const uint32_t row0 = runs.row0[r] + first, h = blockIdx.y;
    __half *dense = (blockIdx.z ? a.vc : a.kc) + (((size_t)runs.seq[r] * a.kv_heads + h) * a.cap + row0) * HD;
    __half *pool = blockIdx.z ? a.vp : a.kp;
    const uint32_t *pages = a.table + (size_t)runs.at[r] * a.max_pages;
    uint4 v[kEach];
    __half *to[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t e = i * kCopyThreads + threadIdx.x, row = e / kChunks, ch = e % kChunks;
        to[i] = nullptr;
        if (row >= rows) continue;
        const uint32_t j = row0 + row, id = pages[j >> a.page_log];
        const bool page = id < a.pages;
        if (!page) atomicOr(a.status, TM_CUDA_STATUS_BAD_PAGE);
        __half *in = dense + (size_t)row * HD + ch * 8u;
        __half *paged = pool + ((((size_t)(page ? id : 0u) * a.kv_heads + h) << a.page_log) + (j & ((1u << a.page_log) - 1u))) * HD + ch * 8u;
        if (TO_PAGES) {
            v[i] = *(const uint4 *)in;
            to[i] = page ? paged : nullptr;
        } else {
            v[i] = page ? *(const uint4 *)paged : make_uint4(0u, 0u, 0u, 0u);
            to[i] = in;
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i)
        if (to[i]) *(uint4 *)to[i] = v[i];
}

// ---- eviction --------------------------------------------------------------------------------------
//
// Per (sequence, KV head): the first `first` rows, the last `recent` rows, and of those between the ones with the largest
// weights, `keep` in all, in their order.  One CTA, or a cluster, finds the smallest weight that stays by counting passes over 11, 11
// and 10 bits of the weights' order-preserving integers, then lists the rows; a second launch moves them.  Up to 4096 rows the
// weights stay in registers, so that a pass is counting alone: 256 heads of up to 4096 rows 13 us.  (Every count adds the
// constant one, which shared memory takes for a whole warp at once whatever the digits: with zeros counted by ballot, so that
// few lanes add to their bin, 14, and with all equal digits of a warp found first 33.)  What bounds the whole: the rows'
// bytes, 8 head_dim each.
constexpr uint32_t kEvictThreads = 512;

struct evict_args {
    __half *kp, *vp;
    const uint32_t *table, *to, *len;
    uint32_t *len_out;  // none where it is `len` itself, which the second launch still reads
    const float *w;
    float *w_out;
    uint32_t *kept, *status;
    uint32_t kv_heads, pages, page_log, max_pages, cap, keep, first, recent;
};

// Weights in order: NaN below everything, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (isnan(w)) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
static_assert(kEvictThreads * 4 == 2048, "four bins a thread");
// Exclusive prefix sum over the CTA's threads, and the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warps, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += up;
    }
    __syncthreads();
    if (lane == 31u) warps[warp] = incl;
    __syncthreads();
    uint32_t w = lane < kEvictThreads / 32u ? warps[lane] : 0u, sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= (uint32_t)o) sum += up;
    }
    total = __shfl_sync(0xffffffffu, sum, 31);
    return __shfl_sync(0xffffffffu, sum - w, warp) + incl - v;
}

constexpr uint32_t kHeld = 8, kStretch = kHeld * kEvictThreads;  // weights of a thread in registers, of a CTA
struct select_smem {
    uint32_t hist[2][2048];
    uint32_t warps[32], found[3];
    uint32_t above, equal;  // rows of this CTA that stay, and at the border
};
template <bool MANY>
__device__ __forceinline__ void sync_all() {
    if (MANY) tmdev::cluster_sync();
    else __syncthreads();
}
__device__ __forceinline__ uint32_t ld_rank(const uint32_t *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tmdev::map_rank(smem_addr(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_rank4(const uint32_t *p, uint32_t rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(tmdev::map_rank(smem_addr(p), rank)) : "memory");
    return v;
}

// Of a head's rows this CTA (`rank` of `ctas` in a cluster; MANY: more than one; a rank behind them has none) looks after
// r0 .. r1.  HELD: their weights stay in registers (at most a stretch of them); else they are read again for every pass, a
// stretch ahead.
constexpr uint32_t kMostCtas = 8;
template <bool HELD, bool MANY>
__device__ __forceinline__ void select_rows(const evict_args &a, const float *w, float *w_out, uint32_t *kept, uint32_t len, uint32_t rank,
                                            uint32_t ctas, select_smem &sm) {
    const uint32_t tid = threadIdx.x;
    const uint32_t per = (len + 16u * ctas - 1u) / (16u * ctas) * 16u, r0 = min(len, rank * per), r1 = min(len, r0 + per);
    const uint32_t lo = a.first, hi = len - a.recent, want = a.keep - a.first - a.recent;
    // (Strips are 4 or 8 rows, whose weights begin on 16 bytes and end within the sequence's: a page has 16 rows or more.)
    const uint32_t strip = HELD && per <= 4u * kEvictThreads ? 4u : 8u, j0 = r0 + tid * strip;
    float held[kHeld];
    auto fetch = [&](float(&v)[kHeld], uint32_t at, uint32_t step) {  // rows at .. at + 3 and, of strips of 8, at + step .. at + step + 3
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e)
            if (4u * e < strip && at + e * step < r1) *(float4 *)&v[4 * e] = *(const float4 *)(w + at + e * step);
    };
    if (HELD) fetch(held, j0, 4u);
    // The want-th largest key between lo and hi, digit by digit: `prefix` its bits so far (those of `mask`), `left` how many
    // are still wanted among the keys that begin with them.
    uint32_t prefix = 0u, mask = 0u, left = want;
    auto equal = [&](uint32_t j, float v) {  // (a row behind r1 has no weight)
        return j >= lo && j < hi && j < r1 && want > 0u && (weight_key(v) & mask) == prefix;
    };
    auto above = [&](uint32_t j, float v) { return j < r1 && (j < lo || j >= hi || (want > 0u && (weight_key(v) & mask) > prefix)); };
    auto in_any_order = [&](auto f) {  // f(row, weight), as it loads best
        fetch(held, r0 + 4u * tid, kStretch / 2);
#pragma unroll 1
        for (uint32_t s0 = r0; s0 < r1; s0 += kStretch) {
            const uint32_t at = s0 + 4u * tid;
            float next[kHeld];
            fetch(next, at + kStretch, kStretch / 2);
#pragma unroll
            for (uint32_t e = 0; e < kHeld; ++e) f(at + e / 4u * (kStretch / 2) + e % 4u, held[e]);
#pragma unroll
            for (uint32_t e = 0; e < kHeld; ++e) held[e] = next[e];
        }
    };
    if (want > 0u) {
        const uint32_t shift[3] = {21u, 10u, 0u}, width[3] = {11u, 11u, 10u};
#pragma unroll 1
        for (uint32_t p = 0; p < 3u; ++p) {
            uint32_t *hist = sm.hist[p & 1u];  // (the other one may still be read by the other CTAs)
            *(uint4 *)(hist + 4u * tid) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            const uint32_t digits = (1u << width[p]) - 1u;
            auto count = [&](uint32_t j, float v) {
                if (equal(j, v)) atomicAdd(&hist[(weight_key(v) >> shift[p]) & digits], 1u);
            };
            if (HELD) {
#pragma unroll
                for (uint32_t e = 0; e < kHeld; ++e)
                    if (e < strip) count(j0 + e, held[e]);
            } else {
                in_any_order(count);
            }
            sync_all<MANY>();
            // Thread i: four bins from 2047 - 4i down, so that a prefix sum counts from the top.
            const uint32_t b = 2044u - 4u * tid;
            uint4 c = *(const uint4 *)(hist + b);
#pragma unroll
            for (uint32_t i = 1; i < (MANY ? kMostCtas : 1u); ++i) {
                const uint32_t of = (rank + i) % kMostCtas;
                if (of >= ctas) continue;
                const uint4 o = ld_rank4(hist + b, of);
                c = make_uint4(c.x + o.x, c.y + o.y, c.z + o.z, c.w + o.w);
            }
            uint32_t total, before = block_scan(c.x + c.y + c.z + c.w, sm.warps, total);
            const uint32_t of[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
            for (uint32_t x = 0; x < 4u; ++x) {
                if (before < left && before + of[x] >= left) {
                    sm.found[0] = b + 3u - x;
                    sm.found[1] = left - before;
                    sm.found[2] = of[x];
                }
                before += of[x];
            }
            __syncthreads();
            prefix |= sm.found[0] << shift[p];
            mask |= digits << shift[p];
            left = sm.found[1];
            if (sm.found[2] == left) break;  // all that begin with these bits stay
        }
    }
    // The rows that stay: those outside lo .. hi and with keys above the border, and the first `left` at it.  Counted and listed
    // stretch by stretch, in order; `stay` and `ties` are those before the stretch.
    uint32_t stay = 0u, ties = 0u, total;
    auto counts = [&](uint32_t s0) {  // of this thread's strip: rows above in the upper half, at the border in the lower
        uint32_t both = 0u;
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e)
            if (e < strip) both += (above(s0 + e, held[e]) ? 1u << 16 : 0u) + (equal(s0 + e, held[e]) ? 1u : 0u);
        return both;
    };
    uint32_t both = 0u;
    if (MANY) {  // what the CTAs before this one have
        if (HELD) {
            both = block_scan(counts(j0), sm.warps, total);
            if (tid == 0) {
                sm.above = total >> 16;
                sm.equal = total & 0xffffu;
            }
        } else {
            uint32_t n_above = 0u, n_equal = 0u;
            in_any_order([&](uint32_t j, float v) {
                n_above += above(j, v) ? 1u : 0u;
                n_equal += equal(j, v) ? 1u : 0u;
            });
            block_scan(n_above, sm.warps, total);
            if (tid == 0) sm.above = total;
            block_scan(n_equal, sm.warps, total);
            if (tid == 0) sm.equal = total;
        }
        tmdev::cluster_sync();  // (all that is HELD has been read)
        for (uint32_t i = 0; i < min(rank, ctas); ++i) {
            stay += ld_rank(&sm.above, i);
            ties += ld_rank(&sm.equal, i);
        }
        if (HELD) tmdev::cluster_arrive();  // nothing of another CTA's is read from here on
    }
#pragma unroll 1
    for (uint32_t s0 = 0; s0 < r1 - r0; s0 += kStretch) {
        if (!HELD) fetch(held, s0 + j0, 4u);
        if (!HELD || !MANY) both = block_scan(counts(s0 + j0), sm.warps, total);  // behind it the stretch's weights are read
        uint32_t n_equal = ties + (both & 0xffffu), at = stay + (both >> 16) + min(n_equal, left);
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e) {
            const uint32_t j = s0 + j0 + e;
            if (e >= strip) continue;
            const bool tie = equal(j, held[e]);
            if (above(j, held[e]) || (tie && n_equal < left)) {
                // what stays moves down, if at all: weights_out may be the weights themselves
                if (HELD || !MANY) w_out[at] = held[e];
                kept[at++] = j;
            }
            n_equal += tie ? 1u : 0u;
        }
        stay += total >> 16;
        ties += total & 0xffffu;
    }
    if (MANY && HELD) tmdev::cluster_wait();
    if (MANY && !HELD) {  // the others may still have to read what this CTA would overwrite: the weights follow together
        tmdev::cluster_sync();
        for (uint32_t i0 = 0; i0 < a.keep; i0 += ctas * kEvictThreads) {
            const uint32_t i = i0 + rank * kEvictThreads + tid;
            const float v = i < a.keep ? w[kept[i]] : 0.0f;
            tmdev::cluster_sync();
            if (i < a.keep) w_out[i] = v;
            tmdev::cluster_sync();
        }
    }
}

// A head's rows are looked after by one CTA, or where there are few heads and a head may have more than a stretch by a cluster.
template <bool MANY>
__global__ void __launch_bounds__(kEvictThreads) kv_evict_select_kernel(const evict_args a) {
    __shared__ __align__(16) select_smem sm;
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t ctas = MANY ? tmdev::cluster_size() : 1u;
    const uint32_t s = blockIdx.y, h = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x, len = a.len[s];
    if (len == kSeqNone || len > a.cap) {
        if (h == 0 && rank == 0 && tid == 0) {
            if (len != kSeqNone) atomicOr(a.status, TM_CUDA_STATUS_PAST_CAPACITY);
            if (a.len_out) a.len_out[s] = len;
        }
        return;
    }
    if (a.len_out && h == 0 && rank == 0 && tid == 0) a.len_out[s] = min(len, a.keep);
    const size_t head = (size_t)s * a.kv_heads + h;
    const float *w = a.w + head * a.cap;
    float *w_out = a.w_out + head * a.cap;
    uint32_t *kept = a.kept + head * a.keep;
    if (len <= a.keep) {
        for (uint32_t i = rank * kEvictThreads + tid; i < a.keep; i += ctas * kEvictThreads) {
            kept[i] = i < len ? i : TM_CUDA_SEQ_NONE;
            if (i < len && w_out != w) w_out[i] = w[i];
        }
        return;
    }
    if (!MANY) {
        if (len <= kStretch) select_rows<true, false>(a, w, w_out, kept, len, 0u, 1u, sm);
        else select_rows<false, false>(a, w, w_out, kept, len, 0u, 1u, sm);
        return;
    }
    // As many as it takes to hold the weights; the others have no rows, but take part in the cluster's barriers.
    const uint32_t need = (len + kStretch - 1u) / kStretch, work = min(ctas, need);
    if (work == 1u) {
        if (rank == 0u) select_rows<true, false>(a, w, w_out, kept, len, 0u, 1u, sm);
    } else if (len <= work * kStretch) select_rows<true, true>(a, w, w_out, kept, len, rank, work, sm);
    else select_rows<false, true>(a, w, w_out, kept, len, rank, work, sm);
}

// Moves the kept rows.
constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kNoRow = 0xffffffffu;  // (a pool has fewer rows than that)

// Row j of a head in the pool, as a number of rows from its start.
__device__ __forceinline__ uint32_t pool_row(const evict_args &a, const uint32_t *pages, uint32_t h, uint32_t j) {
    const uint32_t id = pages[j >> a.page_log];
    if (id < a.pages) return ((id * a.kv_heads + h) << a.page_log) + (j & ((1u << a.page_log) - 1u));
    atomicOr(a.status, TM_CUDA_STATUS_BAD_PAGE);
    return kNoRow;
}

// Into other pages: a CTA takes 16 KB of a head's rows, keys or values.  A row's place is behind two loads that depend on one
// another (its number, its page): a thread a row looks them up, then all copy as in kv_pages_copy_kernel.  Many small CTAs
// hide that better than few that look two stretches ahead (32 sequences of 4096 rows cut to 2048, 493 MB: 76 us, 6.5 TB/s;
// 86 us; 8 KB a CTA 84).
template <int HD>
constexpr uint32_t kRowsMoved = 8192u / HD;
template <int HD>
__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const evict_args a) {
    constexpr uint32_t kMoveRows = kRowsMoved<HD>, kChunks = HD / 8, kEach = kMoveRows * kChunks / kMoveThreads;
    static_assert(kMoveRows <= kMoveThreads, "a thread a row");
    __shared__ uint32_t src[kMoveRows], dst[kMoveRows];
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t s = blockIdx.y / a.kv_heads, h = blockIdx.y % a.kv_heads, len = a.len[s], i0 = blockIdx.x * kMoveRows;
    if (len > a.cap || i0 >= min(len, a.keep)) return;
    const uint32_t rows = min(kMoveRows, min(len, a.keep) - i0);
    if (threadIdx.x < rows) {
        const uint32_t i = i0 + threadIdx.x, j = a.kept[(size_t)blockIdx.y * a.keep + i];
        src[threadIdx.x] = pool_row(a, a.table + (size_t)s * a.max_pages, h, j);
        dst[threadIdx.x] = pool_row(a, a.to + (size_t)s * a.max_pages, h, i);
    }
    __syncthreads();
    __half *pool = blockIdx.z ? a.vp : a.kp;
    uint4 v[kEach];
    uint32_t to[kEach];
#pragma unroll
    for (uint32_t x = 0; x < kEach; ++x) {
        const uint32_t e = x * kMoveThreads + threadIdx.x, row = e / kChunks, from = row < rows ? src[row] : kNoRow;
        to[x] = row < rows ? dst[row] : kNoRow;
        v[x] = from != kNoRow ? *(const uint4 *)(pool + (size_t)from * HD + e % kChunks * 8u) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (uint32_t x = 0; x < kEach; ++x)
        if (to[x] != kNoRow) *(uint4 *)(pool + (size_t)to[x] * HD + (x * kMoveThreads + threadIdx.x) % kChunks * 8u) = v[x];
}

// In place: a CTA takes 64 bytes of every row of a head, so that the columns need not wait for one another, and goes up the
// rows: what it stores lies at or below what it has read.  Bound by the loads' latency, three behind one another a stretch, and with
// few heads by the few CTAs (the whole eviction, 8 heads of 128, in place and into other pages: one sequence of 1001 rows to 300 9.3
// and 7.3 us, of 16000 to 8000 109 and 26, 32 of up to 4096 to 2048 112 and 91).
constexpr uint32_t kShiftEach = 8, kShiftRows = kMoveThreads / 4 * kShiftEach;
template <int HD>
__global__ void __launch_bounds__(kMoveThreads) kv_evict_shift_kernel(const evict_args a) {
    constexpr uint32_t kSlices = HD / 32;
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t s = blockIdx.y / a.kv_heads, h = blockIdx.y % a.kv_heads, len = a.len[s];
    if (len > a.cap || len <= a.keep) return;
    __half *pool = blockIdx.x / kSlices ? a.vp : a.kp;
    const uint32_t *pages = a.table + (size_t)s * a.max_pages, *kept = a.kept + (size_t)blockIdx.y * a.keep;
    const uint32_t r = threadIdx.x / 4u, col = (blockIdx.x % kSlices * 4u + threadIdx.x % 4u) * 8u;
    for (uint32_t i0 = 0; i0 < a.keep; i0 += kShiftRows) {
        uint4 v[kShiftEach];
        uint32_t dst[kShiftEach];
#pragma unroll
        for (uint32_t x = 0; x < kShiftEach; ++x) {
            const uint32_t i = i0 + x * (kMoveThreads / 4) + r;
            dst[x] = kNoRow;
            if (i >= a.keep) continue;
            const uint32_t j = kept[i];
            if (j == i) continue;  // it stays where it is
            const uint32_t src = pool_row(a, pages, h, j);
            dst[x] = pool_row(a, pages, h, i);
            v[x] = src != kNoRow ? *(const uint4 *)(pool + (size_t)src * HD + col) : make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();  // the whole stretch is read
#pragma unroll
        for (uint32_t x = 0; x < kShiftEach; ++x)
            if (dst[x] != kNoRow) *(uint4 *)(pool + (size_t)dst[x] * HD + col) = v[x];
        __syncthreads();  // and written before the next is read
    }
}

// The lengths, where they replace the ones that both launches above read.
__global__ void kv_evict_lengths_kernel(uint32_t *len, uint32_t n_seq, uint32_t keep, uint32_t cap) {
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < n_seq && len[s] <= cap) len[s] = min(len[s], keep);
}

template <int HD>
cudaError_t launch_move(tm_cuda_ctx *ctx, const evict_args &a, uint32_t n_seq, bool in_place) {
    if (in_place)
        return tm_launch_pdl(ctx, kv_evict_shift_kernel<HD>, dim3(2 * (HD / 32), n_seq * a.kv_heads), dim3(kMoveThreads), 0, a);
    return tm_launch_pdl(ctx, kv_evict_move_kernel<HD>, dim3((a.keep + kRowsMoved<HD> - 1) / kRowsMoved<HD>, n_seq * a.kv_heads, 2),
                         dim3(kMoveThreads), 0, a);
}

template <int HD>
cudaError_t launch_copy(tm_cuda_ctx *ctx, const copy_args &a, const copy_runs &runs, bool to_pages) {
    const dim3 grid(runs.tile0[runs.n], a.kv_heads, 2);
    return to_pages ? tm_launch_pdl(ctx, kv_pages_copy_kernel<HD, true>, grid, dim3(kCopyThreads), 0, a, runs)
                    : tm_launch_pdl(ctx, kv_pages_copy_kernel<HD, false>, grid, dim3(kCopyThreads), 0, a, runs);
}

struct pool_shape {
    uint32_t pages, page_rows, max_pages, kv_heads, head_dim;
};
int check_pool(const pool_shape &p, const char *what, char *err, size_t err_cap) {
    if (!pages_ok(p.head_dim, p.page_rows) || p.kv_heads == 0 || p.kv_heads > 4096u || p.pages == 0 || p.max_pages == 0 ||
        (uint64_t)p.max_pages * p.page_rows > 1u << 25 || (uint64_t)p.pages * p.kv_heads * p.page_rows > 0xffffffffu)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS,
                       "%s: head_dim %u (32, 64, 128 or 256), %u KV heads, %u pages of %u rows (16, 32, 64, 128 or 256), %u "
                       "pages a sequence", what, p.head_dim, p.kv_heads, p.pages, p.page_rows, p.max_pages);
    return TM_CUDA_OK;
}
size_t pool_bytes(const pool_shape &p) { return (size_t)p.pages * p.kv_heads * p.page_rows * p.head_dim * 2; }

}  // namespace

extern "C" {

int tm_cuda_kv_pages_supported(uint32_t head_dim, uint32_t page_rows) { return pages_ok(head_dim, page_rows) ? 1 : 0; }

size_t tm_cuda_attention_paged_scratch_bytes(uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                             uint32_t page_rows, uint32_t max_pages, int weights) {
    if (kv_heads == 0 || heads % kv_heads != 0 || !pages_ok(head_dim, page_rows)) return 0;
    return scratch_parts(n_seq, heads, kv_heads, head_dim, (uint64_t)max_pages * page_rows, weights != 0).end;
}

int tm_cuda_attention_decode_paged_dev(tm_cuda_ctx *ctx, tm_cuda_buffer *q, tm_cuda_buffer *k, tm_cuda_buffer *v,
                                       tm_cuda_buffer *q_norm, tm_cuda_buffer *k_norm, tm_cuda_buffer *inv_freq,
                                       tm_cuda_buffer *k_pages, tm_cuda_buffer *v_pages, tm_cuda_buffer *table,
                                       tm_cuda_buffer *out, tm_cuda_buffer *scratch, tm_cuda_buffer *pos_buf,
                                       tm_cuda_buffer *len_buf, tm_cuda_buffer *status, tm_cuda_buffer *weights_in,
                                       tm_cuda_buffer *weights_out, uint32_t n_seq, uint32_t q_stride, uint32_t kv_stride,
                                       uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n_rot,
                                       uint32_t pages, uint32_t page_rows, uint32_t max_pages, uint32_t window, float eps,
                                       float scale, char *err, size_t err_cap) {
    TM_ENTER();
    const pool_shape shape = {pages, page_rows, max_pages, kv_heads, head_dim};
    if (const int rc = check_pool(shape, "paged attention", err, err_cap)) return rc;
    if (heads == 0 || heads % kv_heads != 0 || heads / kv_heads > 32u || n_rot == 0 || n_rot > head_dim || n_rot % 2 != 0)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "paged attention: heads %u/%u (1 to 32 a KV head), n_rot %u of head_dim %u",
                       heads, kv_heads, n_rot, head_dim);
    if (n_seq == 0 || n_seq > TM_CUDA_PAGED_MAX_SEQUENCES)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "sequence count %u outside 1..%u", n_seq, (unsigned)TM_CUDA_PAGED_MAX_SEQUENCES);
    if (weights_in && !weights_out)
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "attention weights are given but not asked for");
    if (q_stride == 0) q_stride = heads * head_dim;
    if (kv_stride == 0) kv_stride = kv_heads * head_dim;
    if (q_stride < heads * head_dim || kv_stride < kv_heads * head_dim)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "row strides %u / %u below the row widths", q_stride, kv_stride);
    if ((uint64_t)n_seq * kv_heads * ((heads / kv_heads + 7u) / 8u) * (((uint64_t)max_pages * page_rows + kTile - 1) / kTile) > 0xffffffffu)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "paged attention: %u sequences of %u KV heads and up to %llu rows", n_seq,
                       kv_heads, (unsigned long long)max_pages * page_rows);
    const size_t nq = ((size_t)(n_seq - 1) * q_stride + (size_t)heads * head_dim) * 4;
    const size_t nkv = ((size_t)(n_seq - 1) * kv_stride + (size_t)kv_heads * head_dim) * 4;
    const size_t cap = (size_t)max_pages * page_rows, nout = (size_t)n_seq * heads * head_dim * 4;
    const size_t nw = (size_t)n_seq * kv_heads * cap * 4, ntable = (size_t)n_seq * max_pages * 4;
    const size_t nscratch = tm_cuda_attention_paged_scratch_bytes(n_seq, heads, kv_heads, head_dim, page_rows, max_pages, weights_out != nullptr);
    TM_CHECK_IN(q, nq, "q");
    TM_CHECK_IN(k, nkv, "k");
    TM_CHECK_IN(v, nkv, "v");
    TM_CHECK_IN(q_norm, (size_t)head_dim * 4, "q norm");
    TM_CHECK_IN(k_norm, (size_t)head_dim * 4, "k norm");
    TM_CHECK_IN(inv_freq, (size_t)(n_rot / 2) * 4, "inv_freq");
    TM_CHECK_BUF(k_pages, pool_bytes(shape), "K pages");
    TM_CHECK_BUF(v_pages, pool_bytes(shape), "V pages");
    TM_CHECK_IN(table, ntable, "page table");
    TM_CHECK_BUF(out, nout, "attention output");
    TM_CHECK_BUF(scratch, nscratch, "paged attention scratch");
    TM_CHECK_IN(pos_buf, (size_t)n_seq * 4, "positions");
    TM_CHECK_IN(len_buf, (size_t)n_seq * 4, "lengths");
    TM_CHECK_BUF(status, 4, "status");
    if (weights_in) TM_CHECK_IN(weights_in, nw, "attention weights");
    if (weights_out) TM_CHECK_BUF(weights_out, nw, "attention weights");
    const tm_span spans[] = {{k_pages, pool_bytes(shape), true, "K pages"}, {v_pages, pool_bytes(shape), true, "V pages"},
                             {out, nout, true, "attention output"}, {scratch, nscratch, true, "scratch"}, {status, 4, true, "status"},
                             {weights_out, nw, true, "attention weights"}, {weights_in, nw, false, "attention weights"},
                             {q, nq, false, "q"}, {k, nkv, false, "k"}, {v, nkv, false, "v"},
                             {q_norm, (size_t)head_dim * 4, false, "q norm"}, {k_norm, (size_t)head_dim * 4, false, "k norm"},
                             {inv_freq, (size_t)(n_rot / 2) * 4, false, "inv_freq"}, {table, ntable, false, "page table"},
                             {pos_buf, (size_t)n_seq * 4, false, "positions"}, {len_buf, (size_t)n_seq * 4, false, "lengths"}};
    if (const int rc = tm_check_disjoint(spans, sizeof spans / sizeof *spans, 5, 6, err, err_cap)) return rc;
    paged_args a = {};
    a.q = (const float *)q->dev;
    a.k = (const float *)k->dev;
    a.v = (const float *)v->dev;
    a.q_norm = (const float *)q_norm->dev;
    a.k_norm = (const float *)k_norm->dev;
    a.inv_freq = (const float *)inv_freq->dev;
    a.kp = (__half *)k_pages->dev;
    a.vp = (__half *)v_pages->dev;
    a.table = (const uint32_t *)table->dev;
    a.pos = (const uint32_t *)pos_buf->dev;
    a.len = (const uint32_t *)len_buf->dev;
    a.out = (float *)out->dev;
    const scratch_parts at(n_seq, heads, kv_heads, head_dim, cap, weights_out != nullptr);
    a.ops = (uint4 *)(scratch->dev + at.ops);
    a.factor = (float *)(scratch->dev + at.factor);
    a.part = (float *)(scratch->dev + at.part);
    a.part_ml = (float2 *)(scratch->dev + at.part_ml);
    a.whole = (float *)(scratch->dev + at.whole);
    a.whole_ml = (float2 *)(scratch->dev + at.whole_ml);
    if (weights_out) {
        a.scores = (float *)(scratch->dev + at.scores);
        a.w_in = weights_in ? (const float *)weights_in->dev : nullptr;
        a.w_out = (float *)weights_out->dev;
    }
    a.status = (uint32_t *)status->dev;
    a.n_seq = n_seq;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    a.blocks = (a.group + 7u) / 8u;
    a.n_rot = n_rot;
    a.pages = pages;
    a.page_log = log2_of(page_rows);
    a.max_pages = max_pages;
    a.cap = (uint32_t)cap;
    a.window = window;
    a.eps = eps;
    a.scale_log2e = scale * 1.4426950408889634f;
    TM_OP_BEGIN("attention_decode_paged");
    TM_CUDA_TRY(head_dim == 32    ? launch_paged<32>(ctx, a)
                : head_dim == 64  ? launch_paged<64>(ctx, a)
                : head_dim == 128 ? launch_paged<128>(ctx, a)
                                  : launch_paged<256>(ctx, a));
    TM_OP_END(3);
}

int tm_cuda_kv_pages_copy_f16(tm_cuda_ctx *ctx, tm_cuda_buffer *k_cache, tm_cuda_buffer *v_cache, tm_cuda_buffer *k_pages,
                              tm_cuda_buffer *v_pages, tm_cuda_buffer *table, tm_cuda_buffer *status, uint32_t pages,
                              uint32_t page_rows, uint32_t max_pages, uint32_t kv_heads, uint32_t head_dim, uint32_t cap,
                              int to_pages, uint32_t n_runs, const uint32_t *runs, char *err, size_t err_cap) {
    TM_ENTER();
    const pool_shape shape = {pages, page_rows, max_pages, kv_heads, head_dim};
    if (const int rc = check_pool(shape, "page copy", err, err_cap)) return rc;
    if (cap == 0 || n_runs == 0 || n_runs > TM_CUDA_PREFILL_SEGMENTS || !runs)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "page copy: capacity %u, %u runs (1 .. %u)", cap, n_runs,
                       (unsigned)TM_CUDA_PREFILL_SEGMENTS);
    copy_runs r;
    r.n = n_runs;
    uint32_t seqs = 0, tables = 0;
    uint64_t tiles = 0;
    for (uint32_t i = 0; i < n_runs; ++i) {
        const uint32_t *p = runs + 4 * (size_t)i;
        if (p[3] == 0 || (uint64_t)p[2] + p[3] > cap || (uint64_t)p[2] + p[3] > (uint64_t)max_pages * page_rows ||
            p[0] > 0xfffffffeu || p[1] > 0xfffffffeu)
            return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "run %u: rows %u..%llu of capacity %u, pages of %llu", i, p[2],
                           (unsigned long long)p[2] + p[3], cap, (unsigned long long)max_pages * page_rows);
        for (uint32_t j = 0; j < i; ++j) {  // two runs store the same row
            const uint32_t *o = runs + 4 * (size_t)j, of = to_pages ? 1 : 0;
            if (o[of] == p[of] && o[2] < p[2] + p[3] && p[2] < o[2] + o[3])
                return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "runs %u and %u store the same rows", j, i);
        }
        r.tile0[i] = (uint32_t)tiles;
        r.seq[i] = p[0];
        r.at[i] = p[1];
        r.row0[i] = p[2];
        r.rows[i] = p[3];
        tiles += (p[3] + kCopyRows - 1) / kCopyRows;
        if (p[0] >= seqs) seqs = p[0] + 1u;
        if (p[1] >= tables) tables = p[1] + 1u;
    }
    if (tiles > 0x7fffffffu) return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "page copy: %llu tiles", (unsigned long long)tiles);
    for (uint32_t i = n_runs; i <= TM_CUDA_PREFILL_SEGMENTS; ++i) r.tile0[i] = (uint32_t)tiles;
    // (128-bit product: sequence numbers are the caller's)
    const unsigned __int128 want = (unsigned __int128)seqs * kv_heads * cap * head_dim * 2;
    if (want > ((unsigned __int128)1 << 62)) return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "page copy: %u dense sequences", seqs);
    const size_t ndense = (size_t)want, ntable = (size_t)tables * max_pages * 4;
    tm_cuda_buffer *const wk = to_pages ? k_pages : k_cache, *const wv = to_pages ? v_pages : v_cache;
    tm_cuda_buffer *const rk = to_pages ? k_cache : k_pages, *const rv = to_pages ? v_cache : v_pages;
    const size_t nw = to_pages ? pool_bytes(shape) : ndense, nr = to_pages ? ndense : pool_bytes(shape);
    TM_CHECK_BUF(wk, nw, to_pages ? "K pages" : "K cache");
    TM_CHECK_BUF(wv, nw, to_pages ? "V pages" : "V cache");
    TM_CHECK_IN(rk, nr, to_pages ? "K cache" : "K pages");
    TM_CHECK_IN(rv, nr, to_pages ? "V cache" : "V pages");
    TM_CHECK_IN(table, ntable, "page table");
    TM_CHECK_BUF(status, 4, "status");
    const tm_span spans[] = {{wk, nw, true, "keys"}, {wv, nw, true, "values"}, {status, 4, true, "status"},
                             {rk, nr, false, "keys"}, {rv, nr, false, "values"}, {table, ntable, false, "page table"}};
    if (const int rc = tm_check_disjoint(spans, sizeof spans / sizeof *spans, 0, 0, err, err_cap)) return rc;
    const copy_args a = {(__half *)k_cache->dev, (__half *)v_cache->dev, (__half *)k_pages->dev, (__half *)v_pages->dev,
                         (const uint32_t *)table->dev, (uint32_t *)status->dev, pages, log2_of(page_rows), max_pages,
                         kv_heads, cap};
    TM_OP_BEGIN("kv_pages_copy");
    TM_CUDA_TRY(head_dim == 32    ? launch_copy<32>(ctx, a, r, to_pages)
                : head_dim == 64  ? launch_copy<64>(ctx, a, r, to_pages)
                : head_dim == 128 ? launch_copy<128>(ctx, a, r, to_pages)
                                  : launch_copy<256>(ctx, a, r, to_pages));
    TM_OP_END(1);
}

int tm_cuda_kv_pages_evict(tm_cuda_ctx *ctx, tm_cuda_buffer *k_pages, tm_cuda_buffer *v_pages, tm_cuda_buffer *table,
                           tm_cuda_buffer *to_table, tm_cuda_buffer *len_buf, tm_cuda_buffer *len_out,
                           tm_cuda_buffer *weights, tm_cuda_buffer *weights_out, tm_cuda_buffer *kept,
                           tm_cuda_buffer *status, uint32_t n_seq, uint32_t kv_heads, uint32_t head_dim, uint32_t pages,
                           uint32_t page_rows, uint32_t max_pages, uint32_t keep, uint32_t first, uint32_t recent, char *err,
                           size_t err_cap) {
    TM_ENTER();
    const pool_shape shape = {pages, page_rows, max_pages, kv_heads, head_dim};
    if (const int rc = check_pool(shape, "eviction", err, err_cap)) return rc;
    const size_t cap = (size_t)max_pages * page_rows;
    if (n_seq == 0 || (uint64_t)n_seq * kv_heads > 65535u)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "eviction: %u sequences of %u KV heads (at most 65535 together)", n_seq, kv_heads);
    if (keep == 0 || keep > cap || (uint64_t)first + recent > keep)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "eviction: keep %u of at most %zu rows, the first %u and the last %u among them",
                       keep, cap, first, recent);
    const size_t nw = (size_t)n_seq * kv_heads * cap * 4, nk = (size_t)n_seq * kv_heads * keep * 4;
    const size_t ntable = (size_t)n_seq * max_pages * 4, nlen = (size_t)n_seq * 4;
    TM_CHECK_BUF(k_pages, pool_bytes(shape), "K pages");
    TM_CHECK_BUF(v_pages, pool_bytes(shape), "V pages");
    TM_CHECK_IN(table, ntable, "page table");
    TM_CHECK_IN(to_table, ntable, "page table to move to");
    TM_CHECK_IN(len_buf, nlen, "lengths");
    TM_CHECK_BUF(len_out, nlen, "new lengths");
    TM_CHECK_IN(weights, nw, "attention weights");
    TM_CHECK_BUF(weights_out, nw, "kept rows' weights");
    TM_CHECK_BUF(kept, nk, "kept rows");
    TM_CHECK_BUF(status, 4, "status");
    const bool same_len = len_out->dev == len_buf->dev;
    const tm_span spans[] = {{k_pages, pool_bytes(shape), true, "K pages"}, {v_pages, pool_bytes(shape), true, "V pages"},
                             {weights_out, nw, true, "kept rows' weights"}, {weights, nw, false, "attention weights"},
                             {kept, nk, true, "kept rows"}, {status, 4, true, "status"}, {table, ntable, false, "page table"},
                             {to_table, ntable, false, "page table to move to"}, {len_out, nlen, true, "new lengths"},
                             {same_len ? nullptr : len_buf, nlen, false, "lengths"}};
    if (const int rc = tm_check_disjoint(spans, sizeof spans / sizeof *spans, 2, 3, err, err_cap)) return rc;
    const bool in_place = to_table->dev == table->dev;
    const evict_args a = {(__half *)k_pages->dev, (__half *)v_pages->dev, (const uint32_t *)table->dev,
                          (const uint32_t *)to_table->dev, (const uint32_t *)len_buf->dev,
                          same_len ? nullptr : (uint32_t *)len_out->dev, (const float *)weights->dev, (float *)weights_out->dev,
                          (uint32_t *)kept->dev, (uint32_t *)status->dev, kv_heads, pages, log2_of(page_rows), max_pages,
                          (uint32_t)cap, keep, first, recent};
    TM_OP_BEGIN("kv_pages_evict");
    // Clusters where the heads leave SMs idle and a head may have more than a CTA's registers hold, of as many CTAs as can have
    // rows (8 KV heads, one sequence of 16000 rows cut to 200, by 4 CTAs a head: 13.3 us, by 8: 17.4, by one 22.8; of 120000 cut to
    // 4000, by 8: 56, by one 150; eight of 16000 cut to 200, by 4: 19.5, by one 27.3).
    const uint64_t heads = (uint64_t)n_seq * kv_heads, room = 2u * (uint32_t)ctx->sm_count;
    uint32_t ctas = 1;
    while (ctas < kMostCtas && ctas * kStretch < cap && 2u * ctas * heads <= room) ctas *= 2;
    const dim3 grid(ctas * kv_heads, n_seq);
    TM_CUDA_TRY(ctas == 1 ? tm_launch_pdl(ctx, kv_evict_select_kernel<false>, grid, dim3(kEvictThreads), 0, a)
                          : tm_launch_cluster_pdl(ctx, ctas, kv_evict_select_kernel<true>, grid, dim3(kEvictThreads), 0, a));
    TM_CUDA_TRY(head_dim == 32    ? launch_move<32>(ctx, a, n_seq, in_place)
                : head_dim == 64  ? launch_move<64>(ctx, a, n_seq, in_place)
                : head_dim == 128 ? launch_move<128>(ctx, a, n_seq, in_place)
                                  : launch_move<256>(ctx, a, n_seq, in_place));
    if (same_len)
        TM_CUDA_TRY(tm_launch_pdl(ctx, kv_evict_lengths_kernel, dim3((n_seq + 127) / 128), dim3(128), 0, (uint32_t *)len_out->dev,
                                  n_seq, keep, (uint32_t)cap));
    TM_OP_END(same_len ? 3 : 2);
}

}  // extern "C"
