// paged_quant_attn.cu — attention of ragged chunks of new tokens over a paged cache held in 8
// bits: the entry point, and which sequences are widened first.
//
// A chunk of many rows reads its keys once for every 256 of them, and the chunk kernel widens
// them as often, while its products read shared memory at the rate that it has: a key tile
// takes it 6,200 clocks and one of 16-bit values 4,000.  So keys of sequences with LONG_ROWS rows and
// more are widened once, into a cache of the workspace, and attended to there
// (8,192 tokens, 32/8 heads of 128, int8: 735 us within the chunk kernel, 494 so, 470 over a 16-bit
// cache, each by itself; in a loop of calls, at the clocks that the power limit leaves, 490-540 and
// 500-530; a key costs 6 KB of memory traffic once, about 1 ns, and 60 ps per head and 256 rows more
// within the kernel: as much at two blocks of eight heads, 512 rows).  The kernels for it cost 25 us
// beside, so a call that cannot come to LONG_TILES products of 256 rows and 128 keys (1.1 us more
// each on one of the SMs, 31 us in all) has none (8 sequences, a chunk of 1,001 tokens among them, a
// window of 1,024: 62 us, 117 widened first).  How long sequences may be is taken from the page table's
// width, so a wide table can bring the launches where nothing is long: 16 sequences' drafted tokens
// over 5,000, 58 us, take 77 with a table for 131,072 tokens and without max_new.  What the workspace
// has no room for stays with the kernels that widen.
#include "paged_rows.cuh"

namespace hmm {
namespace serve {
namespace {

constexpr int LONG_ROWS = 512;
constexpr int64_t LONG_TILES = 4096;
constexpr int WIDE_TOKENS = 128;                     // tokens of a page of the workspace's cache
constexpr int64_t WIDE_BYTES = int64_t(1) << 30;     // of that cache, at most
constexpr int CL_THREADS = 1024, WD_THREADS = 256;

// Whether some sequences may be long, and where they would go.
struct WidePlan {
    int64_t pages, most;     // of the workspace's cache (0: none), and sequences there, at most
    bool all;                // one sequence, which has room: it goes there whatever its rows
    size_t kernels, parts, wide_parts, owner, table, wide_kernels, cache;   // bytes of the workspace's pieces
    size_t bytes() const { return kernels + parts + wide_parts + owner + table + wide_kernels + 2 * cache; }
};

WidePlan wide_plan(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t hk, int64_t D, int64_t max_kv, int64_t window,
                   int64_t max_new, bool shared) {
    WidePlan w{};
    const int64_t group = std::max<int64_t>(1, n_heads / hk), rows = n_tokens * group;
    const int64_t keys = window > 0 ? std::min(max_kv, window + 256) : max_kv;   // of 256 rows, about
    const bool never = n_seq == 0 || (max_new > 0 && std::min(max_new, n_tokens) * group < LONG_ROWS) || rows < LONG_ROWS ||
                       (shared ? 2 : 1) * rows / 256 * hk * ((keys + 127) / 128) < LONG_TILES;
    if (!never) {
        const int64_t per_seq = (max_kv + WIDE_TOKENS - 1) / WIDE_TOKENS;
        w.most = std::min(n_seq, (shared ? 2 : 1) * rows / LONG_ROWS);
        w.pages = std::min(w.most * per_seq, WIDE_BYTES / (4 * WIDE_TOKENS * hk * D));
        w.all = n_seq == 1 && !shared && w.pages >= per_seq;
    }
    w.kernels = up256(attention_workspace(n_seq, n_tokens, n_heads, hk, D, shared || w.pages > 0));
    if (w.pages > 0) {
        w.parts = up256(2 * sizeof(int4) * (size_t)n_seq);
        w.wide_parts = up256(2 * sizeof(int4) * (size_t)w.most);
        w.owner = up256(sizeof(int2) * (size_t)w.pages);
        w.table = up256(sizeof(int32_t) * (size_t)w.pages);
        w.wide_kernels = up256(attention_workspace(w.most, n_tokens, n_heads, hk, D, true));
        w.cache = up256(2 * (size_t)(w.pages * hk * WIDE_TOKENS * D));
    }
    return w;
}

struct WideArgs {
    AttnArgs a;              // the call's
    int4 *parts, *wide;      // [n_seq], [most]: those that stay, those that go
    int2* owner;             // [pages] sequence, page of it; -1: none
    int32_t* table;          // [pages] their numbers
    void *k, *v;             // [pages][hk][WIDE_TOKENS][D]
    int pages, most;
    bool all;
};

// One block.  The long sequences, in order, as long as there is room.
__global__ void __launch_bounds__(CL_THREADS) paged_wide_parts_kernel(const __grid_constant__ WideArgs w) {
    __shared__ int sum[2][CL_THREADS / 32];
    const AttnArgs& a = w.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int p = threadIdx.x; p < w.pages; p += CL_THREADS) {
        w.owner[p] = make_int2(-1, 0);
        w.table[p] = p;
    }
    __syncthreads();
    int base = 0, count = 0;                             // pages and sequences so far
    for (int s0 = 0; s0 < a.b.n_seq; s0 += CL_THREADS) {
        const int s = s0 + threadIdx.x;
        Seq q{};
        if (s < a.b.n_seq) q = load_seq(a.b, a.max_kv, s, a.status);
        const bool is = q.n_new > 0 && (w.all || (int64_t)q.n_new * a.group >= LONG_ROWS);
        int pages = is ? min((q.kv + WIDE_TOKENS - 1) / WIDE_TOKENS, w.pages + 1) : 0, n = is;
        const int own = pages;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {               // (at most 1,024 (pages + 1): in 31 bits)
            const int x = __shfl_up_sync(0xffffffffu, pages, o), y = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) {
                pages += x;
                n += y;
            }
        }
        if (lane == 31) {
            sum[0][warp] = pages;
            sum[1][warp] = n;
        }
        __syncthreads();
        int first = base + pages - own, index = count + n - is;
        for (int i = 0; i < CL_THREADS / 32; ++i) {
            if (i < warp) {
                first += sum[0][i];
                index += sum[1][i];
            }
            base = min(base + sum[0][i], w.pages + 1);   // (no room is no room)
            count += sum[1][i];
        }
        __syncthreads();
        const bool goes = is && index < w.most && first + own <= w.pages;
        if (s < a.b.n_seq) {
            const int4 x = make_int4(q.begin, q.n_new, q.kv, q.pos0);
            w.parts[2 * s] = goes ? make_int4(q.begin, 0, 0, 0) : x;
            w.parts[2 * s + 1] = goes ? make_int4(0, q.row, q.out, 0) : make_int4(q.lo, q.row, q.out, 0);
            if (is && index < w.most) {
                w.wide[2 * index] = goes ? x : make_int4(0, 0, 0, 0);
                w.wide[2 * index + 1] = goes ? make_int4(q.lo, first, q.out, 0) : make_int4(0, 0, 0, 0);
            }
            if (goes)
                for (int i = 0; i < own; ++i) w.owner[first + i] = make_int2(s, i);
        }
    }
    for (int i = count + threadIdx.x; i < w.most; i += CL_THREADS) w.wide[2 * i] = w.wide[2 * i + 1] = make_int4(0, 0, 0, 0);
}

// A block per page and head of the workspace's cache.  Bound by memory: 33 bytes read and 64
// written for 32 values.
template <typename T, int C>
__global__ void __launch_bounds__(WD_THREADS) paged_widen_kernel(const __grid_constant__ WideArgs w) {
    const AttnArgs& a = w.a;
    const int2 own = __ldg(w.owner + blockIdx.x);
    if (own.x < 0) return;
    const Seq q = load_seq(a.b, a.max_kv, own.x, a.status);
    const int kvh = blockIdx.y, key0 = own.y * WIDE_TOKENS;
    // what some row sees: behind the first row's window, and the first tokens
    const int lo = a.window > 0 ? max(0, q.pos0 - a.window + 1) : q.lo;
    if (key0 + WIDE_TOKENS <= lo && key0 >= (a.window > 0 ? a.sinks : 0)) return;
    const int pieces = a.D / 16, all = WIDE_TOKENS * pieces;
    const int64_t to = ((int64_t)blockIdx.x * a.hk + kvh) * WIDE_TOKENS * a.D;
#pragma unroll 2
    for (int i = threadIdx.x; i < all; i += WD_THREADS) {
        const int t = i / pieces, c = i - t * pieces, key = key0 + t;
        if (key >= q.kv || (key < lo && key >= (a.window > 0 ? a.sinks : 0))) continue;
        const KeyRows r = key_rows<C>(a, q.row, kvh, key);
        uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
        uint32_t sx = 127, sy = 127;
        if (r.k) {
            x = __ldg(reinterpret_cast<const uint4*>(r.k) + c);
            y = __ldg(reinterpret_cast<const uint4*>(r.v) + c);
            sx = __ldg(r.ks + (c >> 1));
            sy = __ldg(r.vs + (c >> 1));
        }
        store16<T, C>((T*)w.k + to + (int64_t)t * a.D + 16 * c, x, sx);
        store16<T, C>((T*)w.v + to + (int64_t)t * a.D + 16 * c, y, sy);
    }
}

template <typename T, int C>
hmm_status_t run_quant(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    const WidePlan p = wide_plan(a.b.n_seq, a.b.n_tokens, a.hq, a.hk, a.D, a.max_kv, a.window, max_new, a.b.shared != nullptr);
    if (p.pages == 0) return run_kernels<T, C>(a, max_new, ws, st);
    WideArgs w{};
    unsigned char* at = ws + p.kernels;
    auto piece = [&](size_t bytes) {
        unsigned char* x = at;
        at += bytes;
        return x;
    };
    w.a = a;
    w.parts = (int4*)piece(p.parts);
    w.wide = (int4*)piece(p.wide_parts);
    w.owner = (int2*)piece(p.owner);
    w.table = (int32_t*)piece(p.table);
    unsigned char* wide_ws = piece(p.wide_kernels);
    w.k = piece(p.cache);
    w.v = piece(p.cache);
    w.pages = (int)p.pages;
    w.most = (int)p.most;
    w.all = p.all;
    hmm_status_t s = launch(paged_wide_parts_kernel, dim3(1), CL_THREADS, 0, false, st, "paged_wide_parts_kernel", w);
    if (s != HMM_OK) return s;
    s = launch(paged_widen_kernel<T, C>, dim3((unsigned)p.pages, (unsigned)a.hk), WD_THREADS, 0, false, st,
               "paged_widen_kernel", w);
    if (s != HMM_OK) return s;
    AttnArgs x = a;
    if (!p.all) {
        x.b.shared = w.parts;
        s = run_kernels<T, C>(x, 0, ws, st);
        if (s != HMM_OK) return s;
    }
    x.b.shared = w.wide;
    x.b.n_seq = w.most;
    x.b.table = w.table;
    x.b.pages_per_seq = 1;                               // (a row of the table is a page's number)
    x.k = Pages{(unsigned char*)w.k, 2 * (int64_t)a.hk * WIDE_TOKENS * a.D, 2 * (int64_t)WIDE_TOKENS * a.D, 2 * (int64_t)a.D};
    x.v = x.k;
    x.v.base = (unsigned char*)w.v;
    x.n_pages = w.pages;
    x.page_tokens = WIDE_TOKENS;
    x.by_page = FastDiv::of(WIDE_TOKENS);
    x.min_rows = LONG_ROWS;
    return run_attention<T, CODEC_NONE>(x, 0, wide_ws, st);
}

}  // namespace

template <>
hmm_status_t run_attention<__nv_bfloat16, CODEC_E4M3>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_quant<__nv_bfloat16, CODEC_E4M3>(a, max_new, ws, st);
}
template <>
hmm_status_t run_attention<__half, CODEC_E4M3>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_quant<__half, CODEC_E4M3>(a, max_new, ws, st);
}
template <>
hmm_status_t run_attention<__nv_bfloat16, CODEC_I8>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_quant<__nv_bfloat16, CODEC_I8>(a, max_new, ws, st);
}
template <>
hmm_status_t run_attention<__half, CODEC_I8>(const AttnArgs& a, int max_new, unsigned char* ws, cudaStream_t st) {
    return run_quant<__half, CODEC_I8>(a, max_new, ws, st);
}

size_t quant_attention_workspace(int64_t n_seq, int64_t n_tokens, int64_t n_heads, int64_t n_kv_heads, int64_t D,
                                 int64_t max_kv, int64_t max_new, int64_t window, bool shared) {
    // (a window over everything is none)
    const size_t wide = wide_plan(n_seq, n_tokens, n_heads, n_kv_heads, D, max_kv, window < max_kv ? window : 0, max_new,
                                  shared).bytes();
    return std::max(wide, attention_workspace(n_seq, n_tokens, n_heads, n_kv_heads, D, shared));
}

}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_quant_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_heads,
                                                           int64_t n_kv_heads, int64_t D, int64_t max_kv,
                                                           int64_t max_new) {
    return hmm_paged_quant_window_attention_workspace_size(n_seq, n_tokens, n_heads, n_kv_heads, D, max_kv, max_new, 0);
}

extern "C" size_t hmm_paged_quant_window_attention_workspace_size(int64_t n_seq, int64_t n_tokens, int64_t n_heads,
                                                                  int64_t n_kv_heads, int64_t D, int64_t max_kv,
                                                                  int64_t max_new, int64_t window) {
    if (n_seq < 0 || n_tokens < 0 || n_heads < 1 || n_kv_heads < 1 || D < 1 || D > 256 || max_kv < 0 || max_new < 0 ||
        window < 0)
        return 0;
    return quant_attention_workspace(n_seq, n_tokens, n_heads, n_kv_heads, D, max_kv, max_new, window, false);
}

extern "C" hmm_status_t hmm_paged_quant_attention(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, int dtype,
                                                  const void* q, int64_t q_token, int64_t q_head, int64_t n_heads,
                                                  float scale, int causal, int64_t window, int64_t sinks, int64_t max_new,
                                                  void* out, float* lse, int32_t* device_status, void* workspace,
                                                  size_t workspace_bytes, void* stream) {
    AttnArgs a{};
    hmm_status_t s = check_quant(cache, batch, &a.b, &a.k, &a.v, &a.quant);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(dtype == HMM_DTYPE_BF16 || dtype == HMM_DTYPE_F16,
                "dtype must be HMM_DTYPE_BF16 or HMM_DTYPE_F16, got %d", dtype);
    const size_t need = hmm_paged_quant_window_attention_workspace_size(
        batch->n_seq, batch->n_tokens, n_heads, cache->n_kv_heads, cache->D, batch->pages_per_seq * cache->page_tokens,
        max_new, window);
    bool nothing;
    s = plan_attention({q, q_token, q_head, n_heads, scale, causal, window, sinks, max_new, out, lse, device_status,
                        workspace, workspace_bytes, need}, quant_dims(*cache), batch, true, &a, &nothing);
    if (s != HMM_OK || nothing) return s;
    const int hint = (int)std::min<int64_t>(max_new, INT32_MAX);
    unsigned char* ws = (unsigned char*)workspace;
    const cudaStream_t st = (cudaStream_t)stream;
    if (cache->codes == HMM_DTYPE_E4M3)
        return dtype == HMM_DTYPE_BF16 ? run_attention<__nv_bfloat16, CODEC_E4M3>(a, hint, ws, st)
                                       : run_attention<__half, CODEC_E4M3>(a, hint, ws, st);
    return dtype == HMM_DTYPE_BF16 ? run_attention<__nv_bfloat16, CODEC_I8>(a, hint, ws, st)
                                   : run_attention<__half, CODEC_I8>(a, hint, ws, st);
}
