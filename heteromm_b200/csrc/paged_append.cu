// paged_append.cu — the step before attention over a paged cache of 16-bit values: what the
// calls of both caches check, and the entry point.
#include <algorithm>
#include <cstdlib>

#include "paged_append.cuh"

namespace hmm {
namespace serve {

hmm_status_t check_batch(const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch, Batch* b,
                         Pages* k, Pages* v) {
    HMM_REQUIRE(cache && batch, "null cache or batch");
    HMM_REQUIRE(cache->dtype == HMM_DTYPE_BF16 || cache->dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", (int)cache->dtype);
    HMM_REQUIRE(cache->D >= 8 && cache->D <= 512 && cache->D % 8 == 0,
                "D must be a multiple of 8 in [8, 512], got %lld", (long long)cache->D);
    HMM_REQUIRE(cache->n_kv_heads >= 1 && cache->n_kv_heads <= 65535,
                "n_kv_heads must be in [1, 65535], got %lld", (long long)cache->n_kv_heads);
    HMM_REQUIRE(cache->page_tokens >= 1 && cache->page_tokens < (int64_t(1) << 31),
                "page_tokens must be >= 1");
    HMM_REQUIRE(cache->n_pages >= 0 && cache->n_pages < (int64_t(1) << 31),
                "n_pages must be in [0, 2^31)");
    HMM_REQUIRE(batch->n_seq >= 0 && batch->n_seq <= 65535, "n_seq must be in [0, 65535], got %lld",
                (long long)batch->n_seq);
    HMM_REQUIRE(batch->pages_per_seq >= 0 && batch->pages_per_seq < (int64_t(1) << 31),
                "pages_per_seq must be in [0, 2^31)");
    HMM_REQUIRE(batch->n_tokens >= 0 && batch->n_tokens <= (int64_t(1) << 30),
                "n_tokens must be in [0, 2^30]");
    HMM_REQUIRE(batch->pages_per_seq * cache->page_tokens < (int64_t(1) << 31),
                "pages_per_seq * page_tokens must be < 2^31");
    if (batch->n_seq > 0 && batch->n_tokens > 0) {
        HMM_REQUIRE(batch->cu_new && batch->kv_len, "null cu_new or kv_len");
        HMM_REQUIRE(batch->page_table || batch->pages_per_seq == 0, "null page table");
        HMM_REQUIRE((cache->k && cache->v) || cache->n_pages == 0, "null page array");
    }
    const int64_t st[6] = {cache->k_page, cache->k_head, cache->k_token,
                           cache->v_page, cache->v_head, cache->v_token};
    for (int64_t s : st)
        HMM_REQUIRE(s >= 0 && s % 8 == 0,
                    "cache strides must be multiples of 8 elements, got %lld", (long long)s);
    HMM_REQUIRE(aligned16(cache->k) && aligned16(cache->v), "page arrays must be 16-byte aligned");
    b->table = batch->page_table;
    b->cu = batch->cu_new;
    b->kv_len = batch->kv_len;
    b->n_seq = (int)batch->n_seq;
    b->pages_per_seq = (int)batch->pages_per_seq;
    b->n_tokens = (int)batch->n_tokens;
    *k = Pages{(unsigned char*)cache->k, 2 * cache->k_page, 2 * cache->k_head, 2 * cache->k_token};
    *v = Pages{(unsigned char*)cache->v, 2 * cache->v_page, 2 * cache->v_head, 2 * cache->v_token};
    return HMM_OK;
}

namespace {

// Rows of n tokens as a call lays them out: `bytes` at p + i token + j head.
struct Laid {
    int64_t p, token, head, heads;
    int64_t extent(int64_t bytes) const { return (heads - 1) * head + bytes; }
};

// Whether rows `d` bytes apart share a byte for some pair of n tokens, `token` bytes apart.
bool tokens_meet(int64_t d, int64_t token, int64_t n, int64_t bytes) {
    if (n == 1 || token == 0) return std::abs(d) < bytes;
    const int64_t down = d / token - (d % token < 0), rest = d - down * token;   // d = down * token + rest
    return (rest < bytes && std::abs(down) < n) || (token - rest < bytes && std::abs(down + 1) < n);
}

// Whether a's rows share a byte with b's.  Heads of one projection's tokens (one token
// stride) are told apart; rows of other strides whose ranges overlap are taken to meet.
bool rows_meet(const Laid& a, const Laid& b, int64_t n, int64_t bytes) {
    if (a.heads == 0 || b.heads == 0) return false;
    if (a.p + (n - 1) * a.token + a.extent(bytes) <= b.p || b.p + (n - 1) * b.token + b.extent(bytes) <= a.p)
        return false;
    if (n > 1 && a.token != b.token) return true;
    const int64_t d = b.p - a.p;
    if (n > 1 && a.token > 0) {   // b's heads behind a's, within a token
        const int64_t rest = (d % a.token + a.token) % a.token;
        if (rest >= a.extent(bytes) && rest + b.extent(bytes) <= a.token) return false;
    }
    if (a.heads * b.heads > (1 << 20)) return true;
    for (int64_t i = 0; i < a.heads; ++i)
        for (int64_t j = 0; j < b.heads; ++j)
            if (tokens_meet(d + j * b.head - i * a.head, a.token, n, bytes)) return true;
    return false;
}

// Whether two of a's own rows share a byte.
bool rows_meet_themselves(const Laid& a, int64_t n, int64_t bytes) {
    if (a.heads == 0) return false;
    if ((a.heads == 1 || a.head >= bytes) && (n == 1 || a.token >= a.extent(bytes))) return false;
    if (n > 1 && a.token < bytes) return true;
    for (int64_t j = 1; j < a.heads; ++j)
        if (tokens_meet(j * a.head, a.token, n, bytes)) return true;
    return false;
}

}  // namespace

hmm_status_t plan_append(const AppendCall& c, const hmm_paged_cache_t& dims, const hmm_paged_batch_t* batch, bool quant,
                         AppendArgs* args, int* mode, int* vpl) {
    const auto [q, q_token, q_head, n_heads, k, k_token, k_head, v, v_token, v_head, q_weight, k_weight, weight_dtype,
                eps, rope, n_pos, rotary_dim, interleaved, positions, q_out, out_token, out_head, device_status] = c;
    const hmm_paged_cache_t* cache = &dims;
    AppendArgs& a = *args;
    *vpl = 0;
    HMM_REQUIRE(n_heads >= 0 && n_heads <= 65535, "n_heads must be in [0, 65535], got %lld",
                (long long)n_heads);
    HMM_REQUIRE(device_status, "null device_status");
    HMM_REQUIRE(!rope || (rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= cache->D),
                "rotary_dim must be even and in [2, D], got %lld", (long long)rotary_dim);
    HMM_REQUIRE(!rope || (n_pos >= 0 && n_pos < (int64_t(1) << 31)), "n_pos out of range");
    HMM_REQUIRE(!(q_weight || k_weight) || weight_dtype == HMM_DTYPE_F32 || weight_dtype == cache->dtype,
                "norm weights must be fp32 or of the cache's type");
    HMM_REQUIRE(eps >= 0.0f, "eps must be >= 0");
    if (batch->n_seq == 0 || batch->n_tokens == 0) return HMM_OK;
    HMM_REQUIRE(batch->pages_per_seq > 0, "tokens to append, but no pages in the page table");
    HMM_REQUIRE(k && v && (n_heads == 0 || (q && q_out)), "null q, k, v or q_out");
    HMM_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                    aligned16(q_weight) && aligned16(k_weight) &&
                    (reinterpret_cast<uintptr_t>(rope) & 7) == 0,
                "q, k, v, q_out and the norm weights must be 16-byte aligned, rope 8-byte");
    const int64_t st[8] = {q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head};
    for (int64_t x : st)
        HMM_REQUIRE(x >= 0 && x % 8 == 0, "row strides must be multiples of 8 elements, got %lld",
                    (long long)x);
    if (n_heads > 0) {
        // Warps read rows steps ahead of those that they write, in no order: q_out's rows are
        // q's own, each at its place, or nobody's.
        const int64_t n = batch->n_tokens, bytes = 2 * cache->D;
        const Laid lo{(int64_t)q_out, 2 * out_token, 2 * out_head, n_heads};
        const bool is_q = q_out == q && (n == 1 || out_token == q_token) && (n_heads == 1 || out_head == q_head);
        HMM_REQUIRE(!rows_meet_themselves(lo, n, bytes), "rows of q_out overlap one another");
        HMM_REQUIRE(is_q || !rows_meet(lo, {(int64_t)q, 2 * q_token, 2 * q_head, n_heads}, n, bytes),
                    "q_out overlaps q, and is not q itself");
        HMM_REQUIRE(!rows_meet(lo, {(int64_t)k, 2 * k_token, 2 * k_head, cache->n_kv_heads}, n, bytes) &&
                        !rows_meet(lo, {(int64_t)v, 2 * v_token, 2 * v_head, cache->n_kv_heads}, n, bytes),
                    "q_out overlaps k or v");
    }
    a.q = Rows{(unsigned char*)const_cast<void*>(q), 2 * q_token, 2 * q_head};
    a.k = Rows{(unsigned char*)const_cast<void*>(k), 2 * k_token, 2 * k_head};
    a.v = Rows{(unsigned char*)const_cast<void*>(v), 2 * v_token, 2 * v_head};
    a.out = Rows{(unsigned char*)q_out, 2 * out_token, 2 * out_head};
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    a.w_f32 = weight_dtype == HMM_DTYPE_F32;
    a.rope = rope;
    a.positions = positions;
    a.n_pos = n_pos;
    a.max_kv = batch->pages_per_seq * cache->page_tokens;
    a.n_pages = (int)cache->n_pages;
    a.hq = (int)n_heads;
    a.hk = (int)cache->n_kv_heads;
    a.D = (int)cache->D;
    a.vecs = a.D / 8;
    a.half = rope ? (int)(rotary_dim / 2) : 0;
    a.page_tokens = (int)cache->page_tokens;
    a.eps = eps;
    a.inv_d = 1.0f / (float)a.D;
    a.status = device_status;
    // Two vectors a lane where that pairs a value with its partner in the lane, or leaves
    // no lane idle; else one, with the partner a shuffle away if vectors pair up.
    // (Four neighbouring vectors of a cache in 8 bits have to lie in neighbouring lanes.)
    const bool four = quant && a.vecs == 4;
    const bool lane = rope && !interleaved && 2 * a.half == a.D && a.half % 8 == 0 &&
                      (a.half & (a.half - 1)) == 0 && a.half <= 256 && !four;
    const bool shuffle = rope && !interleaved && !lane && a.half % 8 == 0 && a.vecs <= 32;
    *vpl = !shuffle && !four && (lane || a.vecs % 2 == 0 || a.vecs > 32) ? 2 : 1;
    *mode = !rope ? ROPE_NONE : interleaved ? ROPE_PAIRS : lane ? ROPE_HALVES_LANE
            : shuffle ? ROPE_HALVES : ROPE_HALVES_SMEM;
    while ((*vpl << a.lpr_log2) < a.vecs) ++a.lpr_log2;
    const int n_groups = 32 >> a.lpr_log2;
    a.steps_q = (a.hq + n_groups - 1) / n_groups;
    a.steps_k = (a.hk + n_groups - 1) / n_groups;
    // As many warps as stay on the GPU, each with a list of tokens; few tokens are shared
    // by several warps, down to a step each.
    const int64_t slots = (int64_t)device_sm_count() * ap_minb(quant) * (AP_THREADS / 32);
    const int64_t steps = a.steps_q + 2 * (int64_t)a.steps_k;
    a.parts = (int)std::min(steps, std::max<int64_t>(1, slots / a.b.n_tokens));
    a.tokens_at_once = (int)std::min<int64_t>(a.b.n_tokens, std::max<int64_t>(1, slots / a.parts));
    return HMM_OK;
}

}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" hmm_status_t hmm_paged_kv_append(
    const hmm_paged_cache_t* cache, const hmm_paged_batch_t* batch, const void* q, int64_t q_token,
    int64_t q_head, int64_t n_heads, const void* k, int64_t k_token, int64_t k_head, const void* v,
    int64_t v_token, int64_t v_head, const void* q_weight, const void* k_weight, int weight_dtype,
    float eps, const float* rope, int64_t n_pos, int64_t rotary_dim, int interleaved,
    const int32_t* positions, void* q_out, int64_t out_token, int64_t out_head,
    int32_t* device_status, void* stream) {
    AppendArgs a{};
    hmm_status_t s = check_batch(cache, batch, &a.b, &a.k_pages, &a.v_pages);
    if (s != HMM_OK) return s;
    int mode, vpl;
    s = plan_append({q, q_token, q_head, n_heads, k, k_token, k_head, v, v_token, v_head, q_weight, k_weight, weight_dtype,
                     eps, rope, n_pos, rotary_dim, interleaved, positions, q_out, out_token, out_head, device_status},
                    *cache, batch, false, &a, &mode, &vpl);
    if (s != HMM_OK || vpl == 0) return s;
    const cudaStream_t cs = (cudaStream_t)stream;
    if (cache->dtype == HMM_DTYPE_BF16)
        return vpl == 2 ? launch_append<__nv_bfloat16, 2, CODEC_NONE>(a, mode, cs)
                        : launch_append<__nv_bfloat16, 1, CODEC_NONE>(a, mode, cs);
    return vpl == 2 ? launch_append<__half, 2, CODEC_NONE>(a, mode, cs)
                    : launch_append<__half, 1, CODEC_NONE>(a, mode, cs);
}
