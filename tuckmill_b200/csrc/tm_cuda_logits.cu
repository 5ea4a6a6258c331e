// Logits of a decode step before the next token is chosen: penalties for tokens that the row's log holds, a bias map, a
// grammar's mask, and the greedy choice among what is left.
//
// What bounds it: 8 bytes a logit (read once, written once) and an eighth for the mask.  A CTA takes a stretch of one row
// whose per-token words (how often the log holds the token, which bias entry names it) fit in shared memory, so nothing
// the size of the vocabulary is kept between calls or cleared: the CTA reads the row's whole log (a few kilobytes that the
// row's CTAs share in L2) and counts the tokens of its own stretch with integer atomics, whose order does not matter.  Each
// step of the arithmetic is rounded to f32 by itself, so a choice does not hang on how an expression was contracted.
#include "tm_cuda_internal.cuh"
#include "tm_cuda_device.cuh"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMostChunks = TM_CUDA_LOGITS_PARTIAL_BYTES / 8;

struct logits_args {
    const float *x;
    float *y;
    const uint32_t *log, *pos, *prompt, *bias_ids, *bias_count, *mask;
    const float *penalties, *bias_values;
    unsigned long long *partial;
    uint32_t n, chunk, log_stride, base, bias_cap, mask_words, log_cap;
};

// (value, index) as one integer: larger values first, then lower indices; 0 is no entry.  -0 counts as +0.
__device__ __forceinline__ unsigned long long choice_key(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.0f), k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)k << 32 | (0xffffffffu - i);
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

__global__ void __launch_bounds__(kThreads) logits_adjust_kernel(const logits_args a) {
    extern __shared__ uint32_t words[];  // [chunk] twice the count of generated tokens, + 1 where the prompt holds it
    uint32_t *entry = words + a.chunk;   // [chunk] last bias entry that names the token, from 1
    __shared__ unsigned long long best_of[kThreads / 32];
    tmdev::pdl_trigger();
    tmdev::pdl_wait();
    const uint32_t r = blockIdx.y, c0 = blockIdx.x * a.chunk, m = min(a.chunk, a.n - c0), tid = threadIdx.x;
    for (uint32_t i = tid; i < (a.bias_ids ? 2 : 1) * a.chunk; i += kThreads) words[i] = 0u;
    __syncthreads();
    float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
    if (a.penalties) {
        rep = a.penalties[r * 3];
        presence = a.penalties[r * 3 + 1];
        frequency = a.penalties[r * 3 + 2];
        const uint32_t n = history(a, r), prompt = a.prompt ? a.prompt[r] : 0u;
        const uint32_t *log = a.log + (size_t)r * a.log_stride;
#pragma unroll 4
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t at = log[i] - c0;
            if (at < m) {
                if (i < prompt) atomicOr(&words[at], 1u);
                else atomicAdd(&words[at], 2u);
            }
        }
    }
    if (a.bias_ids) {
        const uint32_t n = min(a.bias_count[r], a.bias_cap);
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t at = a.bias_ids[(size_t)r * a.bias_cap + i] - c0;
            if (at < m) atomicMax(&entry[at], i + 1u);
        }
    }
    __syncthreads();
    const float *x = a.x + (size_t)r * a.n + c0;
    float *y = a.y + (size_t)r * a.n + c0;
    unsigned long long best = 0ull;
    for (uint32_t i = tid; i < m; i += kThreads) {
        float v = x[i];
        const uint32_t word = words[i], count = word >> 1, e = a.bias_ids ? entry[i] : 0u;
        if (word != 0u) v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
        if (count != 0u) v = __fsub_rn(__fsub_rn(v, __fmul_rn(frequency, (float)count)), presence);
        if (e != 0u) v = __fadd_rn(v, a.bias_values[(size_t)r * a.bias_cap + e - 1u]);
        const uint32_t t = c0 + i;
        const bool allowed = !a.mask || (a.mask[(size_t)r * a.mask_words + t / 32u] >> (t & 31u) & 1u);
        if (!allowed) v = -INFINITY;
        y[i] = v;
        if (allowed && !isnan(v)) best = max(best, choice_key(v, t));
    }
    if (!a.partial) return;
    best = warp_max(best);
    if ((tid & 31u) == 0u) best_of[tid >> 5] = best;
    __syncthreads();
    if (tid < 32u) {
        best = warp_max(tid < kThreads / 32 ? best_of[tid] : 0ull);
        if (tid == 0u) a.partial[(size_t)r * kMostChunks + blockIdx.x] = best;
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
        const uint32_t id = best ? 0xffffffffu - (uint32_t)best : 0xffffffffu;
        log[(size_t)r * log_stride + slot] = id;
        if (mirror) mirror[(size_t)r * log_stride + slot] = id;
    }
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
    if (prompt_len && !penalties)
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "prompt lengths are for penalties");
    if (mirror && !partial) return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "a mirror is for a choice");
    if ((bias_ids || bias_values || bias_count) && (!bias_ids || !bias_values || !bias_count || bias_cap == 0))
        return tm_fail(err, err_cap, TM_CUDA_ERR_UNSUPPORTED, "a bias map is ids, values and counts of at most %u entries", bias_cap);
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
    a.log = u32(log);
    a.pos = u32(pos_buf);
    a.prompt = u32(prompt_len);
    a.bias_ids = u32(bias_ids);
    a.bias_count = u32(bias_count);
    a.mask = u32(mask);
    a.penalties = penalties ? (const float *)penalties->dev : nullptr;
    a.bias_values = bias_values ? (const float *)bias_values->dev : nullptr;
    a.partial = partial ? (unsigned long long *)partial->dev : nullptr;
    a.n = n;
    a.chunk = n <= 1024u * kMostChunks ? 1024u : (n + kMostChunks - 1) / kMostChunks;
    a.log_stride = log_stride;
    a.base = base;
    a.bias_cap = bias_cap;
    a.mask_words = words;
    a.log_cap = log_cap;
    const uint32_t chunks = (n + a.chunk - 1) / a.chunk;
    const size_t smem = (size_t)a.chunk * 4 * (bias_ids ? 2 : 1);
    if (smem > 48u * 1024u)  // (more than 1.5 million logits with a bias map: at most 64 KB)
        TM_CUDA_TRY(cudaFuncSetAttribute(logits_adjust_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    TM_OP_BEGIN("logits_adjust_rows");
    TM_CUDA_TRY(tm_launch_pdl(ctx, logits_adjust_kernel, dim3(chunks, n_rows), dim3(kThreads), smem, a));
    if (partial)
        TM_CUDA_TRY(tm_launch_pdl(ctx, logits_choose_kernel, dim3(n_rows), dim3(32), 0, (const unsigned long long *)a.partial,
                                  chunks, (uint32_t *)log->dev, log_stride, base, a.pos, log_cap,
                                  mirror ? (uint32_t *)mirror->dev : nullptr));
    TM_OP_END(partial ? 2 : 1);
}

}  // extern "C"
