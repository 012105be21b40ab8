// paged_pages.cu — page management of a paged cache: copying pages, freeing,
// forking and growing sequences, moving the live pages to the front.
//
// The state is three integer arrays (page table, references, lengths); a call
// reads one state and writes the next one, in place or not.  Two launches for
// a call that allocates:
//   state_pass_kernel  copies the state, and leaves what the second launch
//                      decides by in the workspace: a bitmap of the free pages
//                      with their count per 1,024 pages, and one number per row
//                      (the pages it needs, or -1 for a request it cannot meet)
//   the call's kernel  a block per row or fork; each adds up the numbers of the
//                      rows before it, so it knows its rank among the free
//                      pages, and whether the whole call can be met, without a
//                      grid-wide wait
// so the pages a row gets are the lowest free ones in row order whatever the
// blocks' order, and nothing but reference counts (integers) is added
// atomically.  The integer work is a few loads deep and latency bounds it;
// page data moves once through registers (read + write), which HBM bounds:
// 16 bytes a thread, four loads in flight, 8 blocks per SM.
#include <algorithm>
#include <initializer_list>

#include "paged_serve.cuh"

namespace hmm {
namespace serve {
namespace {

constexpr int PG_THREADS = 256;
constexpr int PG_CHUNK = 1024;             // pages per free count
constexpr int PG_WORDS = PG_CHUNK / 32;
constexpr int PG_VECS = 4;                 // 16-byte loads in flight per thread
constexpr int PG_BLOCKS_PER_SM = 8;
constexpr int PG_BITMAP_WORDS = 48 * 1024; // validation bitmap in shared memory: 1.5 Mi pages a pass

struct State {
    const int32_t *table_in, *refs_in, *kv_in;
    int32_t *table, *refs, *kv;            // the new state
    int n_seq, pps, n_pages, chunks;
};

struct Work {                              // workspace
    int32_t* flags;                        // [0] refused, [1] moved pages
    int32_t* cnt;                          // [chunks] free pages
    uint32_t* bitmap;                      // [chunks * PG_WORDS] free pages
    int32_t* info;                         // [n_seq]
    int32_t* list;                         // [n_pages] free pages by rank; compact: holes
    int32_t* movers;                       // [n_pages]
    uint32_t* map;                         // [n_pages]
};

struct Store {
    unsigned char *k, *v;
    int64_t page_bytes, n_layers, k_page, k_layer, v_page, v_layer;
};

enum Op { OP_COPY_STATE, OP_FORK, OP_GROW };

__device__ __forceinline__ int block_sum(int v, int* sm) {   // every thread gets the sum
    v = __reduce_add_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    int r = 0;
#pragma unroll
    for (int w = 0; w < PG_THREADS / 32; ++w) r += sm[w];
    __syncthreads();
    return r;
}

// Blocks [0, chunks): references.  Blocks [chunks, chunks + n_seq): rows.
template <int OP>
__global__ void __launch_bounds__(PG_THREADS)
state_pass_kernel(const State s, const Work w, int page_tokens, const int32_t* a, const int32_t* b,
                  int n) {
    __shared__ int sm[PG_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && threadIdx.x == 0) w.flags[0] = 0;
    if ((int)blockIdx.x < s.chunks) {
        const int64_t p0 = (int64_t)blockIdx.x * PG_CHUNK;
        int free = 0;
#pragma unroll
        for (int i = 0; i < PG_CHUNK / PG_THREADS; ++i) {
            const int64_t p = p0 + i * PG_THREADS + threadIdx.x;
            const int r = p < s.n_pages ? s.refs_in[p] : 1;
            if (p < s.n_pages && s.refs != s.refs_in) s.refs[p] = r;
            const unsigned m = __ballot_sync(0xffffffffu, r == 0);
            if (lane == 0) w.bitmap[(int64_t)blockIdx.x * PG_WORDS + i * (PG_THREADS / 32) + warp] = m;
            free += r == 0;
        }
        free = block_sum(free, sm);
        if (threadIdx.x == 0) w.cnt[blockIdx.x] = free;
        return;
    }
    const int row = blockIdx.x - s.chunks;
    const int32_t* in = s.table_in + (int64_t)row * s.pps;
    int32_t* out = s.table + (int64_t)row * s.pps;
    const int kv = s.kv_in ? s.kv_in[row] : 0;
    if (threadIdx.x == 0 && s.kv && s.kv != s.kv_in) s.kv[row] = kv;
    const int64_t room = (int64_t)s.pps * page_tokens;
    int64_t lo = 0, hi = 0;      // OP_GROW: entries that the new tokens touch; OP_FORK: that the old ones fill
    bool bad = false, is_src = false, is_dst = false;
    if (OP == OP_GROW) {
        const int64_t add = a[row];
        bad = add < 0 || kv < 0 || kv + add > room;
        if (!bad && add > 0) {
            lo = kv / page_tokens;
            hi = (kv + add + page_tokens - 1) / page_tokens;
        }
    } else if (OP == OP_FORK) {
        int src = 0, dst = 0;
        for (int i = threadIdx.x; i < n; i += PG_THREADS) {
            src += a[i] == row;
            dst += b[i] == row;
        }
        src = block_sum(src, sm);
        dst = block_sum(dst, sm);
        is_src = src > 0;
        is_dst = dst > 0;
        bad = dst > 1 || (is_src && is_dst) || (is_src && (kv < 0 || kv > room)) || (is_dst && kv != 0);
        hi = is_src && !bad ? ((int64_t)kv + page_tokens - 1) / page_tokens : 0;
    }
    int missing = 0, wrong = 0;
    for (int i = threadIdx.x; i < s.pps; i += PG_THREADS) {
        const int e = in[i];
        if (out != in) out[i] = e;
        if (i >= lo && i < hi) {
            missing += e < 0;
            wrong += e >= s.n_pages;
        }
        if (OP == OP_FORK && is_dst) wrong += e >= 0;
    }
    if (OP == OP_COPY_STATE) return;
    missing = block_sum(missing, sm);
    wrong = block_sum(wrong, sm);
    if (threadIdx.x == 0) w.info[row] = bad || wrong ? -1 : OP == OP_GROW ? missing : 0;
}

// The free pages of ranks [base, base + need), lowest first, into list[rank].
// One block; `sm` holds 8 + 256 + 256 words.
__device__ __forceinline__ void emit_free(const Work& w, int chunks, int64_t base, int need, unsigned* sm) {
    unsigned* wt = sm;
    unsigned* pref = sm + 8;
    unsigned* cnt = sm + 8 + PG_THREADS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t run = 0;
    for (int c0 = 0; c0 < chunks && run < base + need; c0 += PG_THREADS) {
        const int c = c0 + threadIdx.x;
        const unsigned v = c < chunks ? (unsigned)w.cnt[c] : 0u;
        const unsigned incl = block_scan_incl_256(v, wt);
        const unsigned total = wt[7];
        pref[threadIdx.x] = incl - v;
        cnt[threadIdx.x] = v;
        __syncthreads();
        if (run + total > base) {
            for (int i = warp; i < PG_THREADS; i += PG_THREADS / 32) {
                const int64_t first = run + pref[i];
                if (cnt[i] == 0 || first >= base + need || first + cnt[i] <= base) continue;
                uint32_t word = w.bitmap[(int64_t)(c0 + i) * PG_WORDS + lane];
                int at = __popc(word);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, at, o);
                    if (lane >= o) at += t;
                }
                int64_t rank = first + at - __popc(word);
                while (word) {
                    const int bit = __ffs(word) - 1;
                    word &= word - 1;
                    if (rank >= base && rank < base + need)
                        w.list[rank] = (c0 + i) * PG_CHUNK + lane * 32 + bit;
                    ++rank;
                }
            }
        }
        run += total;
        __syncthreads();
    }
}

__device__ __forceinline__ int64_t total_free(const Work& w, int chunks, int* sm) {
    int v = 0;   // <= n_pages < 2^31
    for (int c = threadIdx.x; c < chunks; c += PG_THREADS) v += w.cnt[c];
    return block_sum(v, sm);
}

// `bytes` bytes of a page, by one block.
__device__ __forceinline__ void copy_bytes(unsigned char* dst, const unsigned char* src, int64_t bytes) {
    for (int64_t at = 16 * threadIdx.x; at < bytes; at += 16 * PG_THREADS * PG_VECS) {
        uint4 v[PG_VECS];
#pragma unroll
        for (int i = 0; i < PG_VECS; ++i)
            if (at + 16 * PG_THREADS * i < bytes)
                v[i] = *reinterpret_cast<const uint4*>(src + at + 16 * PG_THREADS * i);
#pragma unroll
        for (int i = 0; i < PG_VECS; ++i)
            if (at + 16 * PG_THREADS * i < bytes)
                *reinterpret_cast<uint4*>(dst + at + 16 * PG_THREADS * i) = v[i];
    }
}

// Page data of pairs [0, n): the blocks of the grid take pieces of 16 KiB
// (PG_THREADS x PG_VECS x 16 bytes) of a page of K or V of a layer in turn.
__device__ __forceinline__ void copy_pairs(const Store& p, const int32_t* src, const int32_t* dst,
                                           int64_t n, int64_t block, int64_t blocks) {
    constexpr int64_t PIECE = 16 * PG_THREADS * PG_VECS;
    const int64_t pieces = (p.page_bytes + PIECE - 1) / PIECE;
    const int64_t per_pair = pieces * 2 * p.n_layers;
    for (int64_t i = block; i < n * per_pair; i += blocks) {
        const int64_t pair = i / per_pair, in = i - pair * per_pair;
        const int64_t part = in / pieces, piece = in - part * pieces;
        const int64_t layer = part >> 1;
        const int64_t s = src[pair], d = dst[pair];
        if (s < 0 || d < 0 || s == d) continue;
        unsigned char* base = part & 1 ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
        const int64_t stride = part & 1 ? p.v_page : p.k_page;
        copy_bytes(base + d * stride + piece * PIECE, base + s * stride + piece * PIECE,
                   min(PIECE, p.page_bytes - piece * PIECE));
    }
}

// ------------------------------------------------------------------ copy
// One block: a bitmap of the destinations in shared memory, 1.5 Mi pages at a
// time; a page that is set twice, or is another pair's source, refuses the
// call (the result would depend on the blocks' order).  1,024 pairs: 4 us.
__global__ void __launch_bounds__(1024)
check_pairs_kernel(const int32_t* src, const int32_t* dst, int n, int n_pages, int words, int32_t* refused,
                   int32_t* status) {
    extern __shared__ uint32_t bits[];
    int bad = 0;
    for (int64_t lo = 0; lo < n_pages || lo == 0; lo += (int64_t)words * 32) {
        for (int i = threadIdx.x; i < words; i += blockDim.x) bits[i] = 0;
        __syncthreads();
        const int64_t hi = lo + (int64_t)words * 32;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int s = src[i], d = dst[i];
            if (s < 0 || d < 0) continue;
            if (s >= n_pages || d >= n_pages) bad = 1;
            else if (d >= lo && d < hi && (atomicOr(&bits[(d - lo) >> 5], 1u << ((d - lo) & 31)) >> ((d - lo) & 31)) & 1)
                bad = 1;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int s = src[i], d = dst[i];
            if (s >= 0 && d >= 0 && s != d && s >= lo && s < hi && s < n_pages &&
                (bits[(s - lo) >> 5] >> ((s - lo) & 31)) & 1)
                bad = 1;
        }
        __syncthreads();
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        *refused = bad;
        if (bad) atomicOr(status, HMM_STATUS_BATCH_BOUNDS);
    }
}

__global__ void __launch_bounds__(PG_THREADS)
copy_pages_kernel(const Store p, const int32_t* src, const int32_t* dst, int n, const int32_t* refused) {
    if (*refused) return;
    copy_pairs(p, src, dst, n, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------ free
__global__ void __launch_bounds__(PG_THREADS)
free_rows_kernel(const State s, const int32_t* seqs, int n, int32_t* status) {
    const int row = blockIdx.x;
    int listed = 0, bad = 0;
    for (int i = threadIdx.x; i < n; i += PG_THREADS) {
        const int q = seqs[i];
        listed |= q == row;
        bad |= q < 0 || q >= s.n_seq;
    }
    bad = __syncthreads_or(bad);
    listed = __syncthreads_or(listed);
    if (bad) {
        if (row == 0 && threadIdx.x == 0) atomicOr(status, HMM_STATUS_BATCH_BOUNDS);
        return;
    }
    if (!listed) return;
    int32_t* out = s.table + (int64_t)row * s.pps;   // holds the old row: in place, or copied
    for (int i = threadIdx.x; i < s.pps; i += PG_THREADS) {
        const int e = out[i];
        if (e < 0) continue;
        if (e >= s.n_pages) {
            atomicOr(status, HMM_STATUS_PAGE_BOUNDS);
        } else if (atomicSub(s.refs + e, 1) <= 0) {   // held by a row, but without a reference
            atomicAdd(s.refs + e, 1);
            atomicOr(status, HMM_STATUS_PAGE_BOUNDS);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s.pps; i += PG_THREADS) out[i] = -1;
    if (threadIdx.x == 0) s.kv[row] = 0;
}

// ------------------------------------------------------------------ fork
// Block (fork, part): part 0 writes the row; parts share the copy of the last page.
__global__ void __launch_bounds__(PG_THREADS)
fork_rows_kernel(const State s, const Work w, const Store p, int page_tokens, const int32_t* src,
                 const int32_t* dst, int n, int32_t* status) {
    __shared__ unsigned sm[8 + 2 * PG_THREADS];
    int* red = reinterpret_cast<int*>(sm);
    const int f = blockIdx.x, part = blockIdx.y;
    // every fork's need: the page its last tokens fill partly, if the source holds it
    int before = 0, need = 0, bad = 0;
    for (int i = threadIdx.x; i < n; i += PG_THREADS) {
        const int a = src[i], b = dst[i];
        if (a < 0 || a >= s.n_seq || b < 0 || b >= s.n_seq) {
            bad = 1;
            continue;
        }
        const int kv = s.kv_in[a];
        if (kv < 0 || kv > (int64_t)s.pps * page_tokens) continue;   // info[a] says so
        const int want = kv % page_tokens != 0 &&
                         s.table_in[(int64_t)a * s.pps + kv / page_tokens] >= 0;
        need += want;
        before += want && i < f;
    }
    for (int i = threadIdx.x; i < s.n_seq; i += PG_THREADS) bad |= w.info[i] < 0;
    bad = __syncthreads_or(bad);
    need = block_sum(need, red);
    before = block_sum(before, red);
    const bool short_of = total_free(w, s.chunks, red) < need;
    if (bad || short_of) {
        if (f == 0 && part == 0 && threadIdx.x == 0)
            atomicOr(status, bad ? HMM_STATUS_BATCH_BOUNDS : HMM_STATUS_NO_PAGES);
        return;
    }
    const int a = src[f], b = dst[f];
    const int kv = s.kv_in[a], full = kv / page_tokens;
    const int32_t* from = s.table_in + (int64_t)a * s.pps;
    const int old = kv % page_tokens != 0 ? from[full] : -1;
    int got = -1;
    if (old >= 0) {
        emit_free(w, s.chunks, before, 1, sm);
        __syncthreads();
        got = w.list[before];   // written by this block (and, the same, by the fork's other parts)
    }
    if (part == 0) {
        int32_t* to = s.table + (int64_t)b * s.pps;
        for (int i = threadIdx.x; i < full; i += PG_THREADS) {
            const int e = from[i];
            to[i] = e < 0 ? -1 : e;
            if (e >= 0) atomicAdd(s.refs + e, 1);
        }
        for (int i = full + threadIdx.x; i < s.pps; i += PG_THREADS) to[i] = i == full ? got : -1;
        if (threadIdx.x == 0) {
            s.kv[b] = kv;
            if (got >= 0) s.refs[got] = 1;
        }
    }
    if (got >= 0) {
        const int32_t pair[2] = {old, got};
        copy_pairs(p, pair, pair + 1, 1, part, gridDim.y);
    }
}

// ------------------------------------------------------------------ grow
__global__ void __launch_bounds__(PG_THREADS)
grow_rows_kernel(const State s, const Work w, int page_tokens, const int32_t* n_new, int32_t* status) {
    __shared__ unsigned sm[8 + 2 * PG_THREADS];
    int* red = reinterpret_cast<int*>(sm);
    const int row = blockIdx.x;
    int bad = 0;
    long long before = 0, need = 0;   // 65,535 rows of up to 2^31 entries
    for (int i = threadIdx.x; i < s.n_seq; i += PG_THREADS) {
        const int v = w.info[i];
        bad |= v < 0;
        need += max(v, 0);
        before += i < row ? max(v, 0) : 0;
    }
    bad = __syncthreads_or(bad);
    // (sums by shuffles: 64-bit shared atomics of all threads took 10 us of 21 at 256 sequences)
    __shared__ long long acc[2][PG_THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        need += __shfl_xor_sync(0xffffffffu, need, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if ((threadIdx.x & 31) == 0) {
        acc[0][threadIdx.x >> 5] = need;
        acc[1][threadIdx.x >> 5] = before;
    }
    __syncthreads();
    need = before = 0;
#pragma unroll
    for (int i = 0; i < PG_THREADS / 32; ++i) {
        need += acc[0][i];
        before += acc[1][i];
    }
    const bool short_of = total_free(w, s.chunks, red) < need;
    if (bad || short_of) {
        if (row == 0 && threadIdx.x == 0)
            atomicOr(status, bad ? HMM_STATUS_BATCH_BOUNDS : HMM_STATUS_NO_PAGES);
        return;
    }
    const int mine = w.info[row];
    const int add = n_new[row], kv = s.kv_in[row];
    __syncthreads();   // kv_in may be kv
    if (threadIdx.x == 0) s.kv[row] = kv + add;
    if (mine == 0) return;
    emit_free(w, s.chunks, before, mine, sm);
    __syncthreads();
    const int lo = kv / page_tokens, hi = (int)(((int64_t)kv + add + page_tokens - 1) / page_tokens);
    int32_t* out = s.table + (int64_t)row * s.pps;
    int done = 0;
    for (int i0 = lo; i0 < hi; i0 += PG_THREADS) {
        const int i = i0 + threadIdx.x;
        const unsigned v = i < hi && out[i] < 0;
        const unsigned incl = block_scan_incl_256(v, sm);
        const unsigned total = sm[7];
        if (v) {
            const int page = w.list[before + done + incl - 1];
            out[i] = page;
            s.refs[page] = 1;
        }
        done += total;
        __syncthreads();
    }
}

// --------------------------------------------------------------- compact
// A block per 1,024 pages.  L = live pages; page p stays (map[p] = p), is free
// (map[p] = ~0) or is the k-th live one at or behind L (map[p] = 2^31 + k,
// movers[k] = p); list[k] = the k-th free page before L.
__global__ void __launch_bounds__(PG_THREADS)
compact_plan_kernel(const State s, const Work w, int32_t* out_live) {
    __shared__ int red[PG_THREADS / 32];
    __shared__ unsigned wt[8];
    int all = 0, before = 0;
    for (int c = threadIdx.x; c < s.chunks; c += PG_THREADS) {
        const int v = w.cnt[c];
        all += v;
        before += c < (int)blockIdx.x ? v : 0;
    }
    all = block_sum(all, red);
    before = block_sum(before, red);   // free pages before this chunk
    const int L = s.n_pages - all;
    // free pages before page L: whole chunks, then the words up to L
    int low = 0;
    const int lc = L / PG_CHUNK;
    for (int c = threadIdx.x; c < lc; c += PG_THREADS) low += w.cnt[c];
    if (threadIdx.x < PG_WORDS && lc < s.chunks) {
        const int first = lc * PG_CHUNK + threadIdx.x * 32;
        const uint32_t word = w.bitmap[(int64_t)lc * PG_WORDS + threadIdx.x];
        const int upto = min(max(L - first, 0), 32);
        low += __popc(upto == 32 ? word : word & ((1u << upto) - 1u));
    }
    low = block_sum(low, red);         // = the number of moved pages
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *out_live = L;
        w.flags[1] = low;
    }
    // four neighbouring pages a thread: the scan's order is the pages'
    const int p0 = blockIdx.x * PG_CHUNK + 4 * threadIdx.x;
    const uint32_t bits = (w.bitmap[(int64_t)blockIdx.x * PG_WORDS + threadIdx.x / 8] >> (4 * (threadIdx.x & 7))) & 15u;
    const unsigned n = __popc(bits);
    int rank = before + (int)(block_scan_incl_256(n, wt) - n);   // free pages before p0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int p = p0 + i;
        const bool free = (bits >> i) & 1;
        if (p < s.n_pages) {
            if (free) {
                w.map[p] = 0xffffffffu;
                if (p < L) w.list[rank] = p;
            } else if (p < L) {
                w.map[p] = (uint32_t)p;
            } else {
                const int k = (p - rank) - (L - low);   // live pages before p, less those before L
                w.map[p] = 0x80000000u + (uint32_t)k;
                w.movers[k] = p;
            }
        }
        rank += free;
    }
}

// Blocks [0, n_seq): the rows.  The rest: the moved pages and their references.
__global__ void __launch_bounds__(PG_THREADS)
compact_move_kernel(const State s, const Work w, const Store p, int32_t* status) {
    if ((int)blockIdx.x < s.n_seq) {
        const int64_t row = (int64_t)blockIdx.x * s.pps;
        for (int i = threadIdx.x; i < s.pps; i += PG_THREADS) {
            const int e = s.table[row + i];   // the old row: in place, or copied
            if (e < 0) continue;
            const uint32_t m = e < s.n_pages ? w.map[e] : 0xffffffffu;
            if (m == 0xffffffffu) atomicOr(status, HMM_STATUS_PAGE_BOUNDS);   // no live page: left as it is
            else if (m & 0x80000000u) s.table[row + i] = w.list[m & 0x7fffffffu];
        }
        return;
    }
    const int n = w.flags[1];
    const int64_t block = blockIdx.x - s.n_seq, blocks = gridDim.x - s.n_seq;
    for (int64_t i = block * PG_THREADS + threadIdx.x; i < n; i += blocks * PG_THREADS) {
        const int from = w.movers[i], to = w.list[i];
        s.refs[to] = s.refs[from];
        s.refs[from] = 0;
    }
    copy_pairs(p, w.movers, w.list, n, block, blocks);
}

// ------------------------------------------------------------------ host

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

int64_t chunks_of(int64_t n_pages) { return (n_pages + PG_CHUNK - 1) / PG_CHUNK; }

size_t layout(int64_t n_seq, int64_t n_pages, unsigned char* base, Work* w) {
    const int64_t c = chunks_of(n_pages);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        unsigned char* p = base + at;
        at += up(bytes);
        return p;
    };
    unsigned char* flags = take(8);
    unsigned char* cnt = take(4 * (size_t)c);
    unsigned char* bitmap = take(4 * (size_t)c * PG_WORDS);
    unsigned char* info = take(4 * (size_t)n_seq);
    unsigned char* list = take(4 * (size_t)n_pages);
    unsigned char* movers = take(4 * (size_t)n_pages);
    unsigned char* map = take(4 * (size_t)n_pages);
    if (w)
        *w = Work{(int32_t*)flags, (int32_t*)cnt, (uint32_t*)bitmap, (int32_t*)info,
                  (int32_t*)list, (int32_t*)movers, (uint32_t*)map};
    return at;
}

hmm_status_t check_state(const hmm_paged_state_t* st, bool with_kv, void* ws, size_t ws_bytes,
                         State* s, Work* w) {
    HMM_REQUIRE(st, "null state");
    HMM_REQUIRE(st->n_seq >= 0 && st->n_seq <= 65535, "n_seq must be in [0, 65535], got %lld",
                (long long)st->n_seq);
    HMM_REQUIRE(st->pages_per_seq >= 0 && st->pages_per_seq < (int64_t(1) << 31),
                "pages_per_seq must be in [0, 2^31)");
    HMM_REQUIRE(st->n_pages >= 0 && st->n_pages < (int64_t(1) << 31) - PG_CHUNK,
                "n_pages must be in [0, 2^31 - 1024)");
    HMM_REQUIRE(st->n_seq * st->pages_per_seq == 0 || (st->table_in && st->table_out), "null page table");
    HMM_REQUIRE(st->n_pages == 0 || (st->refs_in && st->refs_out), "null refs");
    HMM_REQUIRE(!with_kv || st->n_seq == 0 || (st->kv_len_in && st->kv_len_out), "null kv_len");
    const size_t need = layout(st->n_seq, st->n_pages, nullptr, nullptr);
    if (!ws || ws_bytes < need)
        return set_error(HMM_ERR_OOM, "workspace too small: %zu < %zu", ws_bytes, need);
    HMM_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 3) == 0, "workspace must be 4-byte aligned");
    layout(st->n_seq, st->n_pages, (unsigned char*)ws, w);
    *s = State{st->table_in, st->refs_in, with_kv ? st->kv_len_in : nullptr,
               st->table_out, st->refs_out, with_kv ? st->kv_len_out : nullptr,
               (int)st->n_seq, (int)st->pages_per_seq, (int)st->n_pages, (int)chunks_of(st->n_pages)};
    return HMM_OK;
}

struct Span {
    const void* p;
    size_t bytes;
    bool meets(const Span& o) const {
        const uintptr_t a = (uintptr_t)p, b = (uintptr_t)o.p;
        return bytes > 0 && o.bytes > 0 && a < b + o.bytes && b < a + bytes;
    }
};

// The last check of a call.  Both launches read the old state and the call's vectors, and
// rely on finding the same: a new array is the old one itself, or apart from all of them
// (`more`: another output, null if there is none).
hmm_status_t check_apart(const State& s, std::initializer_list<Span> read, Span more = {}) {
    const size_t size[3] = {4 * (size_t)s.n_seq * s.pps, 4 * (size_t)s.n_pages, s.kv ? 4 * (size_t)s.n_seq : 0};
    const Span in[3] = {{s.table_in, size[0]}, {s.refs_in, size[1]}, {s.kv_in, size[2]}};
    const Span out[4] = {{s.table, size[0]}, {s.refs, size[1]}, {s.kv, size[2]}, more};
    for (int x = 0; x < 4; ++x) {
        for (int y = 0; y < 3; ++y)
            HMM_REQUIRE(!out[x].meets(in[y]) || (x == y && out[x].p == in[y].p),
                        "a new array overlaps an old one, and is not that one itself");
        for (int y = 0; y < x; ++y) HMM_REQUIRE(!out[x].meets(out[y]), "the new arrays overlap");
        for (const Span& r : read) HMM_REQUIRE(!out[x].meets(r), "a new array overlaps what the call reads");
    }
    return HMM_OK;
}

hmm_status_t check_store(const hmm_page_store_t* st, Store* p) {
    HMM_REQUIRE(st, "null store");
    HMM_REQUIRE(st->n_pages >= 0 && st->n_pages < (int64_t(1) << 31), "n_pages must be in [0, 2^31)");
    HMM_REQUIRE(st->n_layers >= 1 && st->n_layers <= 32767, "n_layers must be in [1, 32767], got %lld",
                (long long)st->n_layers);
    HMM_REQUIRE(st->page_bytes >= 16 && st->page_bytes % 16 == 0,
                "page_bytes must be a positive multiple of 16, got %lld", (long long)st->page_bytes);
    HMM_REQUIRE(st->n_pages == 0 || (st->k && st->v), "null page array");
    HMM_REQUIRE(aligned16(st->k) && aligned16(st->v), "page arrays must be 16-byte aligned");
    const int64_t str[4] = {st->k_page, st->k_layer, st->v_page, st->v_layer};
    for (int64_t x : str)
        HMM_REQUIRE(x >= 0 && x % 16 == 0, "page strides must be multiples of 16 bytes, got %lld",
                    (long long)x);
    HMM_REQUIRE(st->n_pages <= 1 || (st->k_page >= st->page_bytes && st->v_page >= st->page_bytes),
                "pages overlap: page stride < page_bytes");
    *p = Store{(unsigned char*)st->k, (unsigned char*)st->v, st->page_bytes, st->n_layers,
               st->k_page, st->k_layer, st->v_page, st->v_layer};
    return HMM_OK;
}

template <int OP>
hmm_status_t state_pass(const State& s, const Work& w, int64_t page_tokens, const int32_t* a,
                        const int32_t* b, int n, cudaStream_t st) {
    const int grid = s.chunks + s.n_seq;
    if (grid == 0) return HMM_OK;
    state_pass_kernel<OP><<<(unsigned)grid, PG_THREADS, 0, st>>>(s, w, (int)page_tokens, a, b, n);
    return check_launch("state_pass_kernel");
}

// Blocks that move `pairs` pages: as many as pieces, at most what the GPU holds at once.
int64_t copy_blocks(const Store& p, int64_t pairs) {
    const int64_t pieces = (p.page_bytes + 16 * PG_THREADS * PG_VECS - 1) / (16 * PG_THREADS * PG_VECS);
    const int64_t most = (int64_t)device_sm_count() * PG_BLOCKS_PER_SM;
    return std::max<int64_t>(1, pairs >= most ? most : std::min(most, pairs * pieces * 2 * p.n_layers));
}

}  // namespace
}  // namespace serve
}  // namespace hmm

using namespace hmm;
using namespace hmm::serve;

extern "C" size_t hmm_paged_state_workspace_size(int64_t n_seq, int64_t n_pages) {
    if (n_seq < 0 || n_pages < 0) return 0;
    return layout(n_seq, n_pages, nullptr, nullptr);
}

extern "C" hmm_status_t hmm_paged_copy_pages(const hmm_page_store_t* store, const int32_t* src,
                                             const int32_t* dst, int64_t n, int32_t* device_status,
                                             void* workspace, size_t workspace_bytes, void* stream) {
    Store p;
    hmm_status_t s = check_store(store, &p);
    if (s != HMM_OK) return s;
    HMM_REQUIRE(n >= 0 && n < (int64_t(1) << 31), "n must be in [0, 2^31), got %lld", (long long)n);
    HMM_REQUIRE(device_status, "null device_status");
    if (n == 0) return HMM_OK;
    HMM_REQUIRE(src && dst, "null src or dst");
    if (!workspace || workspace_bytes < 4)
        return set_error(HMM_ERR_OOM, "workspace too small: %zu < 4", workspace_bytes);
    const cudaStream_t st = (cudaStream_t)stream;
    const int64_t words = std::min<int64_t>(PG_BITMAP_WORDS, std::max<int64_t>(1, (store->n_pages + 31) / 32));
    static std::atomic<uint64_t> done{0};
    s = allow_smem(check_pairs_kernel, PG_BITMAP_WORDS * 4, &done);
    if (s != HMM_OK) return s;
    int32_t* refused = (int32_t*)workspace;
    check_pairs_kernel<<<1, 1024, words * 4, st>>>(src, dst, (int)n, (int)store->n_pages, (int)words,
                                                   refused, device_status);
    s = check_launch("check_pairs_kernel");
    if (s != HMM_OK) return s;
    copy_pages_kernel<<<(unsigned)copy_blocks(p, n), PG_THREADS, 0, st>>>(p, src, dst, (int)n, refused);
    return check_launch("copy_pages_kernel");
}

extern "C" hmm_status_t hmm_paged_free(const hmm_paged_state_t* state, const int32_t* seqs, int64_t n,
                                       int32_t* device_status, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    State s;
    Work w;
    hmm_status_t e = check_state(state, true, workspace, workspace_bytes, &s, &w);
    if (e != HMM_OK) return e;
    HMM_REQUIRE(n >= 0 && n < (int64_t(1) << 31), "n must be in [0, 2^31), got %lld", (long long)n);
    HMM_REQUIRE(device_status && (n == 0 || seqs), "null seqs or device_status");
    e = check_apart(s, {{seqs, 4 * (size_t)n}});
    if (e != HMM_OK) return e;
    const cudaStream_t st = (cudaStream_t)stream;
    if (s.table != s.table_in || s.refs != s.refs_in || s.kv != s.kv_in) {
        e = state_pass<OP_COPY_STATE>(s, w, 1, nullptr, nullptr, 0, st);
        if (e != HMM_OK) return e;
    }
    if (n == 0 || s.n_seq == 0) return HMM_OK;
    free_rows_kernel<<<(unsigned)s.n_seq, PG_THREADS, 0, st>>>(s, seqs, (int)n, device_status);
    return check_launch("free_rows_kernel");
}

extern "C" hmm_status_t hmm_paged_fork(const hmm_paged_state_t* state, const hmm_page_store_t* store,
                                       int64_t page_tokens, const int32_t* src, const int32_t* dst,
                                       int64_t n, int32_t* device_status, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    State s;
    Work w;
    Store p;
    hmm_status_t e = check_state(state, true, workspace, workspace_bytes, &s, &w);
    if (e != HMM_OK) return e;
    e = check_store(store, &p);
    if (e != HMM_OK) return e;
    HMM_REQUIRE(store->n_pages == state->n_pages, "the store has %lld pages, the state %lld",
                (long long)store->n_pages, (long long)state->n_pages);
    HMM_REQUIRE(page_tokens >= 1 && page_tokens < (int64_t(1) << 31) &&
                    state->pages_per_seq * page_tokens < (int64_t(1) << 31),
                "page_tokens must be >= 1 and pages_per_seq * page_tokens < 2^31");
    HMM_REQUIRE(n >= 0 && n <= 65535, "n must be in [0, 65535], got %lld", (long long)n);
    HMM_REQUIRE(device_status && (n == 0 || (src && dst)), "null src, dst or device_status");
    e = check_apart(s, {{src, 4 * (size_t)n}, {dst, 4 * (size_t)n}});
    if (e != HMM_OK) return e;
    const cudaStream_t st = (cudaStream_t)stream;
    e = state_pass<OP_FORK>(s, w, page_tokens, src, dst, (int)n, st);
    if (e != HMM_OK || n == 0) return e;
    const int64_t parts = std::min<int64_t>(copy_blocks(p, 1), 64);
    fork_rows_kernel<<<dim3((unsigned)n, (unsigned)parts), PG_THREADS, 0, st>>>(
        s, w, p, (int)page_tokens, src, dst, (int)n, device_status);
    return check_launch("fork_rows_kernel");
}

extern "C" hmm_status_t hmm_paged_grow(const hmm_paged_state_t* state, int64_t page_tokens,
                                       const int32_t* n_new, int32_t* device_status, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    State s;
    Work w;
    hmm_status_t e = check_state(state, true, workspace, workspace_bytes, &s, &w);
    if (e != HMM_OK) return e;
    HMM_REQUIRE(page_tokens >= 1 && page_tokens < (int64_t(1) << 31) &&
                    state->pages_per_seq * page_tokens < (int64_t(1) << 31),
                "page_tokens must be >= 1 and pages_per_seq * page_tokens < 2^31");
    HMM_REQUIRE(device_status && (s.n_seq == 0 || n_new), "null n_new or device_status");
    // (lengths that double in place: a row's block reads its own number, then writes it)
    const bool doubles = n_new == s.kv && s.kv == s.kv_in;
    e = check_apart(s, {{n_new, doubles ? 0 : 4 * (size_t)s.n_seq}});
    if (e != HMM_OK) return e;
    const cudaStream_t st = (cudaStream_t)stream;
    e = state_pass<OP_GROW>(s, w, page_tokens, n_new, nullptr, 0, st);
    if (e != HMM_OK || s.n_seq == 0) return e;
    grow_rows_kernel<<<(unsigned)s.n_seq, PG_THREADS, 0, st>>>(s, w, (int)page_tokens, n_new, device_status);
    return check_launch("grow_rows_kernel");
}

extern "C" hmm_status_t hmm_paged_compact(const hmm_paged_state_t* state, const hmm_page_store_t* store,
                                          int32_t* out_live, int32_t* device_status, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    State s;
    Work w;
    Store p;
    hmm_status_t e = check_state(state, false, workspace, workspace_bytes, &s, &w);
    if (e != HMM_OK) return e;
    e = check_store(store, &p);
    if (e != HMM_OK) return e;
    HMM_REQUIRE(store->n_pages == state->n_pages, "the store has %lld pages, the state %lld",
                (long long)store->n_pages, (long long)state->n_pages);
    HMM_REQUIRE(out_live && device_status, "null out_live or device_status");
    e = check_apart(s, {}, {out_live, 4});
    if (e != HMM_OK) return e;
    const cudaStream_t st = (cudaStream_t)stream;
    if (s.n_pages == 0) {
        HMM_CUDA_TRY(cudaMemsetAsync(out_live, 0, sizeof(int32_t), st));
        return state_pass<OP_COPY_STATE>(s, w, 1, nullptr, nullptr, 0, st);
    }
    e = state_pass<OP_COPY_STATE>(s, w, 1, nullptr, nullptr, 0, st);
    if (e != HMM_OK) return e;
    compact_plan_kernel<<<(unsigned)s.chunks, PG_THREADS, 0, st>>>(s, w, out_live);
    e = check_launch("compact_plan_kernel");
    if (e != HMM_OK) return e;
    const unsigned grid = (unsigned)(s.n_seq + copy_blocks(p, (s.n_pages + 1) / 2));
    compact_move_kernel<<<grid, PG_THREADS, 0, st>>>(s, w, p, device_status);
    return check_launch("compact_move_kernel");
}
