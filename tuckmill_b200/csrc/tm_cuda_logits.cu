// Logits of a decode step before the next token is chosen: penalties for tokens that the row's log holds, a bias map, a
// grammar's mask, and the greedy choice among what is left.
//
// What bounds it: 8 bytes a logit (read once, written once) and an eighth for the mask.  A CTA takes a stretch of one row
// whose per-token words fit in shared memory, so nothing the size of the vocabulary is kept between calls or cleared: the
// CTA reads the row's whole log and bias map (a few kilobytes that the row's CTAs share in L2) and counts the tokens of its
// own stretch with integer atomics, whose order does not matter, while its logits are on their way into registers.  The
// arithmetic is done once for each named token; all other logits pass from registers to memory under the mask (words tested
// for every logit: 32 rows of 151936 34 us instead of 17.3; the log read once by a cluster of CTAs that send each other its
// entries: 19.4; mask and bits worked out for a whole word by one lane, fewer instructions, for which all wait: 17.1, and 25.7
// instead of 25.1 for 48 rows of 262144).  Each step is rounded to f32 by itself, so a choice does not hang on how an
// expression was contracted.
#include "tm_cuda_internal.cuh"
#include "tm_cuda_device.cuh"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kCountBits = 20;
static_assert(TM_CUDA_LOGITS_MAX_LOG < 1u << kCountBits && TM_CUDA_LOGITS_MAX_BIASES < 1u << (32 - kCountBits), "fit in a token's word");
constexpr uint32_t kMostChunks = TM_CUDA_LOGITS_PARTIAL_BYTES / 8, kNone = 0xffffffffu;

struct logits_args {
    const float *x;
    float *y;
    const uint32_t *log, *pos, *prompt, *bias_ids, *bias_count, *mask;
    const float *penalties, *bias_values;
    unsigned long long *partial;
    uint32_t n, log_stride, base, bias_cap, mask_words, log_cap;
    bool quads;  // rows of x and y begin on 16 bytes
};

// Floats as integers in their order; -0 counts as +0, nothing but NaN maps to 0 .. 0x7fffff.  A (value, index) pair is one
// integer, larger values first, then lower indices; 0 is no pair.
__device__ __forceinline__ uint32_t order(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// Entries of row r's log before the slot that is chosen now.
__device__ __forceinline__ uint32_t history(const logits_args &a, uint32_t r) {
    return (uint32_t)min((uint64_t)a.base + a.pos[r], (uint64_t)a.log_cap);
}

// The best of a warp's (value, index) pairs, as the first lane's key.
__device__ __forceinline__ unsigned long long warp_best(float v, uint32_t at) {
    const uint32_t k = at == kNone ? 0u : order(v), top = __reduce_max_sync(0xffffffffu, k);
    const uint32_t low = __reduce_min_sync(0xffffffffu, k == top ? at : kNone);
    return top == 0u ? 0ull : (unsigned long long)top << 32 | (0xffffffffu - low);
}

// EACH quads of logits a thread: a stretch of EACH * 1024 logits.
template <int EACH>
__global__ void __launch_bounds__(kThreads, EACH == 8 ? 4 : 5) logits_adjust_kernel(const logits_args a) {
    constexpr uint32_t kChunk = EACH * 4u * kThreads, kBatch = 8;
    constexpr int kHalf = EACH > 4 ? 4 : EACH;  // quads that are on their way while the log is counted
    // Of each token: how often the log holds it from the prompt's end on, and above those bits its last bias entry, from 1.
    __shared__ __align__(16) uint32_t words[kChunk];
    __shared__ uint32_t logged[kChunk / 32], biased[kChunk / 32];  // a bit a token: the log holds it; the bias map names it
    __shared__ unsigned long long keys[kThreads / 32];
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t r = blockIdx.y, c0 = blockIdx.x * kChunk, m = min(kChunk, a.n - c0), tid = threadIdx.x;
    const float *x = a.x + (size_t)r * a.n + c0;
    float *y = a.y + (size_t)r * a.n + c0;
    const uint32_t *mask = a.mask ? a.mask + (size_t)r * a.mask_words + c0 / 32u : nullptr;
    const uint32_t *log = a.log + (size_t)r * a.log_stride, *ids = a.bias_ids + (size_t)r * a.bias_cap;
    // The first entries of the log and of the bias map are asked for before the row's lengths have arrived.
    uint32_t log_id[kBatch], bias_id = a.bias_ids && tid < a.bias_cap ? ids[tid] : kNone;
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) log_id[u] = a.penalties && u * kThreads + tid < a.log_cap ? log[u * kThreads + tid] : kNone;
    const uint32_t n_log = a.penalties ? history(a, r) : 0u, prompt = a.penalties && a.prompt ? a.prompt[r] : 0u;
    const uint32_t n_bias = a.bias_ids ? min(a.bias_count[r], a.bias_cap) : 0u;
    float v[EACH][4];
    uint32_t allowed = 0u;  // a bit a logit of this thread: the mask lets it through
    auto fetch = [&](int e) {
        const uint32_t i = (e * kThreads + tid) * 4u;
        if (a.quads) {
            if (i < m) *(float4 *)v[e] = *(const float4 *)(x + i);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[e][k] = i + k < m ? x[i + k] : 0.0f;
        }
    };
#pragma unroll
    for (int e = 0; e < kHalf; ++e) fetch(e);
    const bool any = a.penalties || a.bias_ids;
    if (any) {
        for (uint32_t i = tid * 4u; i < kChunk; i += kThreads * 4u) *(uint4 *)(words + i) = make_uint4(0u, 0u, 0u, 0u);
        for (uint32_t i = tid; i < kChunk / 32; i += kThreads) logged[i] = biased[i] = 0u;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const uint32_t i = (e * kThreads + tid) * 4u;
        if (i < m) allowed |= ((mask ? mask[i / 32u] >> (i & 31u) : 15u) & 15u) << (4 * e);
    }
    if (any) {
        __syncthreads();
        if (a.bias_ids) {
            for (uint32_t i = tid; i < n_bias; i += kThreads) {
                const uint32_t at = (i == tid ? bias_id : ids[i]) - c0;
                if (at >= m) continue;
                atomicOr(&biased[at / 32u], 1u << (at & 31u));
                atomicMax(&words[at], (i + 1u) << kCountBits);
            }
            __syncthreads();
        }
        for (uint32_t i0 = tid; i0 < n_log; i0 += kBatch * kThreads) {  // kBatch loads on their way at a time
            if (i0 != tid) {
#pragma unroll
                for (uint32_t u = 0; u < kBatch; ++u) log_id[u] = i0 + u * kThreads < n_log ? log[i0 + u * kThreads] : kNone;
            }
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                const uint32_t at = log_id[u] - c0, i = i0 + u * kThreads;
                if (at < m && i < n_log) {
                    atomicOr(&logged[at / 32u], 1u << (at & 31u));
                    if (i >= prompt) atomicAdd(&words[at], 1u);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = kHalf; e < EACH; ++e) fetch(e);
    // ---- the logits that nothing names; the others are stored as they are ----
    float best = -INFINITY;
    // The best's quad; a bit a logit of this thread: a candidate here, named.
    uint32_t best_quad = 0u, mine = 0u, others = 0u;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const uint32_t i = (e * kThreads + tid) * 4u;
        if (i >= m) continue;
        const uint32_t in = m - i < 4u ? (1u << (m - i)) - 1u : 15u, named = any ? (logged[i / 32u] | biased[i / 32u]) >> (i & 31u) & in : 0u;
        const uint32_t let = allowed >> (4 * e), can = let & ~named & in, show = let | named;
        mine |= can << (4 * e);
        others |= named << (4 * e);
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            top = fmaxf(top, can >> k & 1u ? v[e][k] : -INFINITY);  // (a NaN is passed over)
            v[e][k] = show >> k & 1u ? v[e][k] : -INFINITY;
        }
        if (top > best) {
            best = top;
            best_quad = e;
        }
        if (a.quads) {
            *(float4 *)(y + i) = *(const float4 *)v[e];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < m) y[i + k] = v[e][k];
        }
    }
    uint32_t best_at = kNone;
    if (a.partial && mine != 0u) {
        if (best > -INFINITY) {
            float q[4];
            uint32_t of = 0u;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (best_quad != e) continue;
                of = mine >> (4 * e);
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = v[e][k];
            }
#pragma unroll
            for (int k = 3; k >= 0; --k)
                if (q[k] == best && (of >> k & 1u) != 0u) best_at = c0 + (best_quad * kThreads + tid) * 4u + k;
        } else {  // the first that is -infinity and no NaN
#pragma unroll
            for (int e = EACH - 1; e >= 0; --e)
#pragma unroll
                for (int k = 3; k >= 0; --k)
                    if (v[e][k] == best && (mine >> (4 * e + k) & 1u) != 0u) best_at = c0 + (e * kThreads + tid) * 4u + k;
        }
    }
    // ---- the others ----
    const float repetition = a.penalties ? a.penalties[r * 3] : 1.0f, presence = a.penalties ? a.penalties[r * 3 + 1] : 0.0f;
    const float frequency = a.penalties ? a.penalties[r * 3 + 2] : 0.0f;
#pragma unroll 1
    for (; others != 0u; others &= others - 1u) {
        const uint32_t j = __ffs(others) - 1u, at = ((j >> 2) * kThreads + tid) * 4u + (j & 3u);
        float z = x[at];  // (this thread has stored it as it was, if y is x)
        const uint32_t word = words[at], count = word & ((1u << kCountBits) - 1u), entry = word >> kCountBits;
        const float bias = entry != 0u ? a.bias_values[(size_t)r * a.bias_cap + entry - 1u] : 0.0f;
        if (logged[at / 32u] >> (at & 31u) & 1u) {
            z = z > 0.0f ? __fdiv_rn(z, repetition) : __fmul_rn(z, repetition);
            if (count != 0u) z = __fsub_rn(__fsub_rn(z, __fmul_rn(frequency, (float)count)), presence);
        }
        if (entry != 0u) z = __fadd_rn(z, bias);
        const bool can = (allowed >> j & 1u) != 0u;
        y[at] = can ? z : -INFINITY;
        if (can && !isnan(z) && (best_at == kNone || z > best || (z == best && c0 + at < best_at))) {
            best = z;
            best_at = c0 + at;
        }
    }
    if (!a.partial || m == 0u) return;
    const unsigned long long key = warp_best(best, best_at);
    if ((tid & 31u) == 0u) keys[tid >> 5] = key;
    __syncthreads();
    if (tid < 32u) {
        const unsigned long long top = warp_max(tid < kThreads / 32 ? keys[tid] : 0ull);
        if (tid == 0u) a.partial[(size_t)r * kMostChunks + blockIdx.x] = top;
    }
}

// A warp per row: the best of its stretches, into the row's log.
__global__ void __launch_bounds__(32) logits_choose_kernel(const unsigned long long *partial, uint32_t chunks, uint32_t *log,
                                                           uint32_t log_stride, uint32_t base, const uint32_t *pos,
                                                           uint32_t log_cap, uint32_t *mirror) {
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t r = blockIdx.x;
    unsigned long long best = 0ull;
    for (uint32_t i = threadIdx.x; i < chunks; i += 32u) best = max(best, partial[(size_t)r * kMostChunks + i]);
    best = warp_max(best);
    const uint64_t slot = (uint64_t)base + pos[r];
    if (threadIdx.x == 0 && slot < log_cap) {
        const uint32_t id = best ? 0xffffffffu - (uint32_t)best : kNone;
        log[(size_t)r * log_stride + slot] = id;
        if (mirror) mirror[(size_t)r * log_stride + slot] = id;
    }
}

template <int EACH>
cudaError_t launch_adjust(tm_cuda_ctx *ctx, const logits_args &a, uint32_t chunks, uint32_t n_rows) {
    return tm_launch_pdl(ctx, logits_adjust_kernel<EACH>, dim3(chunks, n_rows), dim3(kThreads), 0, a);
}

}  // namespace

extern "C" {

int tm_cuda_logits_adjust_rows_f32_dev(tm_cuda_ctx *ctx, tm_cuda_buffer *x, tm_cuda_buffer *y, uint32_t n_rows, uint32_t n,
                                       tm_cuda_buffer *log, uint32_t log_stride, uint32_t base, tm_cuda_buffer *pos_buf,
                                       uint32_t log_cap, tm_cuda_buffer *prompt_len, tm_cuda_buffer *penalties,
                                       tm_cuda_buffer *bias_ids, tm_cuda_buffer *bias_values, tm_cuda_buffer *bias_count,
                                       uint32_t bias_cap, tm_cuda_buffer *mask, tm_cuda_buffer *partial,
                                       tm_cuda_buffer *mirror, char *err, size_t err_cap) {
    TM_ENTER();
    if (n == 0 || n > TM_CUDA_LOGITS_MAX || n_rows == 0 || n_rows > 65535u)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "%u rows (1 .. 65535) of %u logits (1 .. %u)", n_rows, n,
                       (unsigned)TM_CUDA_LOGITS_MAX);
    const bool uses_log = penalties || partial;
    if (uses_log && (!log || !pos_buf))
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "penalties and a choice need the token logs and positions");
    if (uses_log && (log_cap == 0 || log_cap > log_stride))
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "token log of %u slots in rows of %u", log_cap, log_stride);
    if (penalties && log_cap > TM_CUDA_LOGITS_MAX_LOG)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "penalties over token logs of %u slots (at most %u)", log_cap, (unsigned)TM_CUDA_LOGITS_MAX_LOG);
    if (prompt_len && !penalties)
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "prompt lengths are for penalties");
    if (mirror && !partial) return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "a mirror is for a choice");
    if ((bias_ids || bias_values || bias_count) && (!bias_ids || !bias_values || !bias_count || bias_cap == 0))
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "a bias map is ids, values and counts of at most %u entries", bias_cap);
    if (bias_ids && bias_cap > TM_CUDA_LOGITS_MAX_BIASES)
        return tm_fail(err, err_cap, TM_CUDA_ERR_BOUNDS, "bias maps of %u entries (at most %u)", bias_cap, (unsigned)TM_CUDA_LOGITS_MAX_BIASES);
    const uint32_t words = (n + 31u) / 32u;
    const size_t nx = (size_t)n_rows * n * 4, nlog = ((size_t)(n_rows - 1) * log_stride + log_cap) * 4, nr = (size_t)n_rows * 4;
    const size_t nbias = (size_t)n_rows * bias_cap * 4, nmask = (size_t)n_rows * words * 4;
    const size_t npart = (size_t)n_rows * TM_CUDA_LOGITS_PARTIAL_BYTES;
    TM_CHECK_IN(x, nx, "logits");
    TM_CHECK_BUF(y, nx, "adjusted logits");
    if (uses_log) {
        if (partial) TM_CHECK_BUF(log, nlog, "token logs");
        else TM_CHECK_IN(log, nlog, "token logs");
        TM_CHECK_IN(pos_buf, nr, "positions");
    } else {  // a handle that is not looked at has to be one all the same
        if (log) TM_CHECK_IN(log, 1, "token logs");
        if (pos_buf) TM_CHECK_IN(pos_buf, 1, "positions");
    }
    if (penalties) TM_CHECK_IN(penalties, nr * 3, "penalties");
    if (prompt_len) TM_CHECK_IN(prompt_len, nr, "prompt lengths");
    if (bias_ids) {
        TM_CHECK_IN(bias_ids, nbias, "bias ids");
        TM_CHECK_IN(bias_values, nbias, "bias values");
        TM_CHECK_IN(bias_count, nr, "bias counts");
    }
    if (mask) TM_CHECK_IN(mask, nmask, "token mask");
    if (partial) TM_CHECK_BUF(partial, npart, "choice partials");
    if (mirror) TM_CHECK_BUF(mirror, nlog, "token log mirrors");
    const tm_span spans[] = {{x, nx, false, "logits"}, {y, nx, true, "adjusted logits"},
                             {uses_log ? log : nullptr, nlog, partial != nullptr, "token logs"},
                             {uses_log ? pos_buf : nullptr, nr, false, "positions"}, {penalties, nr * 3, false, "penalties"},
                             {prompt_len, nr, false, "prompt lengths"}, {bias_ids, nbias, false, "bias ids"},
                             {bias_values, nbias, false, "bias values"}, {bias_count, nr, false, "bias counts"},
                             {mask, nmask, false, "token mask"}, {partial, npart, true, "choice partials"},
                             {mirror, nlog, true, "token log mirrors"}};
    if (const int rc = tm_check_disjoint(spans, sizeof spans / sizeof *spans, 0, 1, err, err_cap)) return rc;
    logits_args a = {};
    auto u32 = [](tm_cuda_buffer *b) { return b ? (const uint32_t *)b->dev : nullptr; };
    a.x = (const float *)x->dev;
    a.y = (float *)y->dev;
    a.log = u32(uses_log ? log : nullptr);
    a.pos = u32(uses_log ? pos_buf : nullptr);
    a.prompt = u32(prompt_len);
    a.bias_ids = u32(bias_ids);
    a.bias_count = u32(bias_count);
    a.mask = u32(mask);
    a.penalties = penalties ? (const float *)penalties->dev : nullptr;
    a.bias_values = bias_values ? (const float *)bias_values->dev : nullptr;
    a.partial = partial ? (unsigned long long *)partial->dev : nullptr;
    a.n = n;
    a.quads = n % 4u == 0u && (((size_t)x->dev | (size_t)y->dev) & 15u) == 0u;
    a.log_stride = log_stride;
    a.base = base;
    a.bias_cap = bias_cap;
    a.mask_words = words;
    a.log_cap = log_cap;
    // Short stretches keep every SM busy with few rows (one of 151936 logits, a log of 600, 1024 logits: 4.3 us), as long as all
    // find a place at once (8 rows, 2048 logits 8.1 us, 4096 9.1; 16 rows, 4096 11.0, 8192 13.4); with many rows long ones,
    // because every CTA reads the row's log (32 rows, logs up to 4000, a mask and a bias map: 4096 logits 18.2, 8192 17.3; 48 of
    // 262144, logs up to 1200: 29, 25.1, floor 15.7).
    const uint32_t sms = (uint32_t)ctx->sm_count;
    uint32_t each = 1;
    while (each < 8u && ((n + each * 1024u - 1) / (each * 1024u) > kMostChunks || (uint64_t)n_rows * ((n + each * 1024u - 1) / (each * 1024u)) > 5u * sms))
        each *= 2;
    const uint32_t chunks = (n + each * 1024u - 1) / (each * 1024u);
    TM_OP_BEGIN("logits_adjust_rows");
    TM_CUDA_TRY(each == 1   ? launch_adjust<1>(ctx, a, chunks, n_rows)
                : each == 2 ? launch_adjust<2>(ctx, a, chunks, n_rows)
                : each == 4 ? launch_adjust<4>(ctx, a, chunks, n_rows)
                            : launch_adjust<8>(ctx, a, chunks, n_rows));
    if (partial)
        TM_CUDA_TRY(tm_launch_pdl(ctx, logits_choose_kernel, dim3(n_rows), dim3(32), 0, (const unsigned long long *)a.partial,
                                  chunks, (uint32_t *)log->dev, log_stride, base, a.pos, log_cap,
                                  mirror ? (uint32_t *)mirror->dev : nullptr));
    TM_OP_END(partial ? 2 : 1);
}

}  // extern "C"
