// Page and slot bookkeeping of a step on the GPU: pages, slots, positions and ancestor masks of the step's tokens from the
// requests' lengths (pkv_plan_step), sequences cut to given lengths (pkv_truncate), and the move of an accepted draft path's
// rows behind the cached tokens (pkv_keep_rows).
//
// All three are latency: a few KB of integers, or the rows of a handful of tokens. So one launch each, no intermediate
// arrays in global memory, and every round trip counts. Results do not depend on the order in which CTAs run: pages are
// handed out in the order of the sequences. Measured, plan and truncate together: 64 sequences, a token each: 11 us; 96 trees of up to
// 32 tokens: 13 us; 48 prompts, 200 000 tokens: 12 us (17 with a token per thread). Rows kept in one layer: 8 us, in eight layers of 48
// sequences: 9.5 us (15 with the rows of a unit one after the other).
#include "pkv_common.cuh"

int pkv_check_cache(const pkv_cache_t* c);

namespace {

constexpr int NT = 1024;
constexpr int MAX_BATCH = 4096;                      // two prefix sums of the batch in static shared memory
constexpr int FILL = 4 * NT;                         // tokens per CTA before another CTA joins: four per thread

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + PKV_PAGE_TOKENS - 1) / PKV_PAGE_TOKENS; }

// the last index s with sums[s] <= i, for ascending sums[0 .. n]; empty entries (equal neighbours) are skipped
__device__ __forceinline__ int owner_of(const int* sums, int n, int i) {
    int lo = 0, hi = n;                              // sums[lo] <= i < sums[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// Exclusive sums of a pair per thread over the block (one barrier pair); the totals are added to `run`, which every
// thread carries from one group of NT entries to the next. 64 bits: a caller's lengths may be anything.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long (&run)[2], long long (*warp_sums)[2], int entries) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 31) { warp_sums[warp][0] = a; warp_sums[warp][1] = b; }
    __syncthreads();
    long long before_a = run[0], before_b = run[1];
#pragma unroll 1
    for (int w = 0; w < (min(entries, NT) + 31) / 32; ++w) {           // (the other warps have none)
        const long long x = warp_sums[w][0], y = warp_sums[w][1];
        if (w < warp) { before_a += x; before_b += y; }
        run[0] += x; run[1] += y;
    }
    __syncthreads();
    a += before_a - a0;
    b += before_b - b0;
}

struct PlanArgs {
    pkv_pages_t pg;
    pkv_plan_t plan;
    const int32_t* n_new;
    const int32_t* parents;
};

// Every CTA forms the same two prefix sums (tokens, new pages) and the same verdict from them, then fills its share of the
// tokens. The k-th new page of the step is free[count - k], so a token's slot is known before the table entry is
// written; the CTA that finishes last writes the tables (the others still read them).
__global__ void __launch_bounds__(NT) pkv_plan_step_kernel(const PlanArgs A) {
    __shared__ int cu_s[MAX_BATCH + 1], off_s[MAX_BATCH + 1];
    __shared__ long long warp_sums[NT / 32][2];
    __shared__ int last_s;
    const int tid = threadIdx.x, B = A.pg.batch, max_pages = A.pg.max_pages, n_pages = A.pg.n_pages;
    int32_t* const table = A.pg.page_table_dev;
    int32_t* const seqlens = A.pg.seqlens_dev;
    int32_t* const pool = A.pg.free_dev;
    const bool tree = A.parents != nullptr;
    pkv_grid_launch_dependents();
    pkv_grid_wait();

    const int count = pool ? min(max(pool[0], 0), n_pages) : 0;
    long long run[2] = {0, 0};
    int bad = 0, where = 0;
    for (int b0 = 0; b0 < B; b0 += NT) {
        const int b = b0 + tid;
        long long n = 0, pages = 0;
        if (b < B) {
            const int L = seqlens[b], m = A.n_new[b];
            if (m < 0 || L < 0 || (long long)L + m > (long long)max_pages * PKV_PAGE_TOKENS || (tree && m > PKV_TREE_MAX)) {
                bad = 4; where = b;
            } else {
                n = m;
                if (pool) pages = pages_of(L + m) - pages_of(L);
            }
        }
        block_scan2(n, pages, run, warp_sums, B - b0);
        if (b < B) {                                 // (sums past 2^31 are refused below, before anyone uses them)
            cu_s[b] = (int)n;
            off_s[b] = (int)pages;
        }
    }
    if (run[0] > A.plan.capacity) { bad = 4; where = -1; }
    if (run[1] > count) { bad = 5; where = (int)min(run[1] - count, 0x7fffffffLL); }
    if (tid == 0) { cu_s[B] = (int)run[0]; off_s[B] = (int)run[1]; }
    bool refused = __syncthreads_or(bad) != 0;
    const int total = refused ? 0 : (int)run[0];
    if (tree && !refused) {                          // a parent comes before its child
        for (int i = tid; i < total; i += NT) {
            const int b = owner_of(cu_s, B, i), p = A.parents[i];
            if (p < -1 || p >= i - cu_s[b]) { bad = 4; where = b; }
        }
        refused = __syncthreads_or(bad) != 0;
    }
    if (bad && blockIdx.x == 0) pkv_report(A.plan.status_dev, bad, where);

    // Four tokens per thread, stored as one vector each where the arrays allow it: mostly of one sequence and page, so one search,
    // one length and one page index serve them.
    const bool wide = ((((uintptr_t)A.plan.slots_dev) | ((uintptr_t)A.plan.seq_dev) | ((uintptr_t)A.plan.positions_dev)) & 15u) == 0;
    for (int i0 = (blockIdx.x * NT + tid) * 4; i0 < A.plan.capacity; i0 += gridDim.x * NT * 4) {
        int slot[4], seq[4], pos[4];
        int b = -1, L = 0, had = 0, at = -1, page = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = i0 + e;
            slot[e] = -1;                            // no token here: a slot that every writer skips
            if (refused || i >= total) continue;
            if (b < 0 || i >= cu_s[b + 1]) {
                b = owner_of(cu_s, B, i);
                L = seqlens[b];
                had = pages_of(L);
                at = -1;
            }
            const int row = i - cu_s[b], t = L + row, p = t / PKV_PAGE_TOKENS;
            if (p != at) {
                at = p;
                if (pool && p >= had) page = pool[count - (off_s[b] + p - had)];
                else page = table[(size_t)b * max_pages + p];
            }
            seq[e] = b;
            if (page >= 0 && page < n_pages) slot[e] = page * PKV_PAGE_TOKENS + t % PKV_PAGE_TOKENS;
            pos[e] = t;
            if (tree) {
                const int32_t* parents = A.parents + cu_s[b];
                unsigned long long word = 0;
                int depth = -1;
                for (int j = row; j >= 0; j = parents[j]) {      // strictly downwards, as checked above
                    word |= 1ull << j;
                    ++depth;
                }
                pos[e] = L + depth;
                A.plan.mask_dev[i] = (int64_t)word;
            } else if (A.plan.mask_dev) {            // a chain: the step's tokens up to this one (words of an earlier tree must not stay)
                A.plan.mask_dev[i] = (int64_t)(row >= PKV_TREE_MAX - 1 ? ~0ull : (2ull << row) - 1);
            }
        }
        if (wide && !refused && i0 + 4 <= total) {
            *reinterpret_cast<int4*>(A.plan.slots_dev + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(A.plan.seq_dev + i0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
            *reinterpret_cast<int4*>(A.plan.positions_dev + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i0 + e >= A.plan.capacity) break;
                A.plan.slots_dev[i0 + e] = slot[e];
                if (!refused && i0 + e < total) { A.plan.seq_dev[i0 + e] = seq[e]; A.plan.positions_dev[i0 + e] = pos[e]; }
            }
        }
    }
    if (blockIdx.x == 0)
        for (int b = tid; b <= B; b += NT) A.plan.cu_dev[b] = refused ? 0 : cu_s[b];
    if (refused) return;

    if (gridDim.x > 1) {
        __syncthreads();                             // this CTA's reads of the tables are done
        if (tid == 0) {
            __threadfence();
            const bool last = atomicAdd(A.plan.ticket_dev, 1u) == gridDim.x - 1;
            if (last) *A.plan.ticket_dev = 0u;       // ready for the next step
            last_s = last;
        }
        __syncthreads();
        if (!last_s) return;
        __threadfence();
    }
    for (int k = tid; k < off_s[B]; k += NT) {       // (no page pool: none)
        const int b = owner_of(off_s, B, k);
        table[(size_t)b * max_pages + pages_of(seqlens[b]) + k - off_s[b]] = pool[count - k];
    }
    __syncthreads();
    for (int b = tid; b < B; b += NT) seqlens[b] += cu_s[b + 1] - cu_s[b];
    if (tid == 0 && pool) pool[0] = count - off_s[B];
}

// One CTA: the pages past the kept length go back to the pool in the reverse of the order in which pkv_plan_step takes them,
// so that a step that is planned and dropped leaves the stack as it was.
__global__ void __launch_bounds__(NT) pkv_truncate_kernel(const pkv_pages_t pg, const int32_t* __restrict__ lengths,
                                                          int32_t* __restrict__ status) {
    __shared__ int off_s[MAX_BATCH + 1];
    __shared__ long long warp_sums[NT / 32][2];
    const int tid = threadIdx.x, B = pg.batch;
    pkv_grid_launch_dependents();
    pkv_grid_wait();
    const int count = pg.free_dev ? min(max(pg.free_dev[0], 0), pg.n_pages) : 0;
    long long run[2] = {0, 0};
    int bad = 0, where = 0;
    for (int b0 = 0; b0 < B; b0 += NT) {
        const int b = b0 + tid;
        long long gone = 0, none = 0;
        if (b < B) {
            const int L = pg.seqlens_dev[b], keep = lengths[b];
            if (keep < 0 || L < 0 || L > pg.max_pages * PKV_PAGE_TOKENS) { bad = 4; where = b; }
            else if (pg.free_dev && keep < L) gone = pages_of(L) - pages_of(keep);
        }
        block_scan2(gone, none, run, warp_sums, B - b0);
        if (b < B) off_s[b] = (int)gone;
    }
    if (tid == 0) off_s[B] = (int)run[0];
    if (run[0] > pg.n_pages - count) { bad = 5; where = -1; }       // more pages than the pool ever held
    const bool refused = __syncthreads_or(bad) != 0;
    if (bad) pkv_report(status, bad, where);
    if (refused) return;
    const int K = (int)run[0];
    for (int k = tid; k < K; k += NT) {
        const int b = owner_of(off_s, B, k);
        int32_t* entry = pg.page_table_dev + (size_t)b * pg.max_pages + pages_of(lengths[b]) + k - off_s[b];
        pg.free_dev[count + K - k] = *entry;
        *entry = -1;
    }
    __syncthreads();
    for (int b = tid; b < B; b += NT) pg.seqlens_dev[b] = min(pg.seqlens_dev[b], lengths[b]);
    if (tid == 0 && pg.free_dev) pg.free_dev[0] = count + K;
}

// ------------------------------------------------------------------------------------------------ accepted rows
constexpr int KC = 32, KR = 8, KT = KC * KR;         // threads of a CTA: column units of a row x groups of rows
constexpr int MAX_LAYERS = 48;                       // layers per launch (their pools are kernel arguments)
constexpr int DEEP = PKV_TREE_MAX / KR;              // rows per thread, all in flight

struct KeepLayer {
    uint8_t* latent;
    uint8_t* v;                                      // bf16 or quantised value pool, or null
    int W, n_kv, head_dim, v_bits;
};
struct KeepArgs {
    KeepLayer layer[MAX_LAYERS];
    pkv_pages_t pg;
    const int32_t *cu, *keep, *n_keep;
    int capacity;
    int32_t* lengths_out;
    int32_t* status;
};

__host__ __device__ inline int keep_units(int W, int n_kv, int head_dim, int v_bits, bool with_v) {
    const int lat = pkv_row_bytes(W) / 16 + pkv_padded_width(W) / 64;
    return lat + (!with_v ? 0 : v_bits ? n_kv * 5 : n_kv * (head_dim / 8));
}

// CTA (32 column units, sequence, layer); a unit is 16 bytes of a row (or the few bytes of its scales). All rows of the units are
// read before any is written: a row's target is another one's source.
__global__ void __launch_bounds__(KT) pkv_keep_rows_kernel(const KeepArgs A) {
    __shared__ int2 moves[PKV_TREE_MAX];
    __shared__ int n_moves;
    const int tid = threadIdx.x, b = blockIdx.y;
    const KeepLayer& Y = A.layer[blockIdx.z];
    pkv_grid_launch_dependents();
    pkv_grid_wait();
    const int lo = A.cu[b], hi = A.cu[b + 1], L = A.pg.seqlens_dev[b], nk = A.n_keep[b], n = hi - lo, base = L - n;
    bool ok = lo >= 0 && hi >= lo && hi <= A.capacity && base >= 0 && L <= A.pg.max_pages * PKV_PAGE_TOKENS && nk >= 0 && nk <= n && nk <= PKV_TREE_MAX;
    if (tid == 0) n_moves = 0;
    __syncthreads();
    if (ok && tid < nk) {
        const int i = A.keep[lo + tid], before = tid ? A.keep[lo + tid - 1] : -1;
        ok = i > before && i < n && i >= 0;
        if (ok) {
            const int s = base + i, d = base + tid;
            const int sp = A.pg.page_table_dev[(size_t)b * A.pg.max_pages + s / PKV_PAGE_TOKENS];
            const int dp = A.pg.page_table_dev[(size_t)b * A.pg.max_pages + d / PKV_PAGE_TOKENS];
            ok = sp >= 0 && sp < A.pg.n_pages && dp >= 0 && dp < A.pg.n_pages;
            moves[tid] = make_int2(sp * PKV_PAGE_TOKENS + s % PKV_PAGE_TOKENS, dp * PKV_PAGE_TOKENS + d % PKV_PAGE_TOKENS);
            if (i != tid) atomicMax(&n_moves, tid + 1);
        }
    }
    const bool refused = __syncthreads_or(!ok) != 0;
    if (blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) {
        if (refused) pkv_report(A.status, 4, b);
        if (A.lengths_out) A.lengths_out[b] = refused ? L : base + nk;
    }
    if (refused || n_moves == 0) return;
    const int RB = pkv_row_bytes(Y.W), nc = RB / 16, ns = pkv_padded_width(Y.W) / 64;
    int u = blockIdx.x * KC + tid % KC, size = 16, g = 0;
    // what unit u is: codes of the latent, four of its block scales, bf16 values, value codes, or a value scale
    int kind = 5;
    uint8_t* pool = Y.latent;
    size_t page_bytes = pkv_page_bytes(Y.W);
    if (u < nc) {
        kind = 0;
    } else if ((u -= nc) < ns) {
        kind = 1; size = 4;
    } else if (Y.v) {
        u -= ns;
        pool = Y.v;
        const int per = Y.v_bits ? 4 : Y.head_dim / 8;
        page_bytes = Y.v_bits ? (size_t)Y.n_kv * PKV_VQ_TILE_BYTES : (size_t)Y.n_kv * PKV_PAGE_TOKENS * Y.head_dim * 2;
        g = u / per;
        if (g < Y.n_kv) { kind = Y.v_bits ? 3 : 2; u %= per; }
        else if (Y.v_bits && (g = u - Y.n_kv * 4) < Y.n_kv) { kind = 4; size = 2; }
    }
    auto at = [&](int slot) -> uint8_t* {
        const uint32_t r = slot % PKV_PAGE_TOKENS;
        const uint32_t o = kind == 0   ? pkv_code_offset(r, u * 16, RB)
                           : kind == 1 ? PKV_PAGE_TOKENS * RB + pkv_scale_offset(r, u * 4)
                           : kind == 2 ? ((uint32_t)g * PKV_PAGE_TOKENS + r) * Y.head_dim * 2 + u * 16
                           : kind == 3 ? (uint32_t)g * 8192 + r * 64 + ((u ^ ((r >> 1) & 3u)) << 4)
                                       : (uint32_t)Y.n_kv * 8192 + g * 256 + r * 2;
        return pool + (size_t)(slot / PKV_PAGE_TOKENS) * page_bytes + o;
    };
    const int n_rows = kind < 5 ? n_moves : 0;
    uint4 val[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        const int j = tid / KC + k * KR;
        if (j >= n_rows) continue;
        const uint8_t* src = at(moves[j].x);
        if (size == 16) val[k] = *reinterpret_cast<const uint4*>(src);
        else if (size == 4) val[k].x = *reinterpret_cast<const uint32_t*>(src);
        else val[k].x = *reinterpret_cast<const uint16_t*>(src);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        const int j = tid / KC + k * KR;
        if (j >= n_rows) continue;
        uint8_t* dst = at(moves[j].y);
        if (size == 16) *reinterpret_cast<uint4*>(dst) = val[k];
        else if (size == 4) *reinterpret_cast<uint32_t*>(dst) = val[k].x;
        else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)val[k].x;
    }
}

int check_pages(const pkv_pages_t* p) {
    if (!p || !p->page_table_dev || !p->seqlens_dev || p->batch < 0 || p->max_pages <= 0 || p->n_pages <= 0) return PKV_ERR_INVALID;
    if (p->batch > MAX_BATCH || p->n_pages > 0x7fffffff / PKV_PAGE_TOKENS || p->max_pages > 0x7fffffff / PKV_PAGE_TOKENS - 1) return PKV_ERR_UNSUPPORTED;
    return PKV_OK;
}

// An array that a call only reads must not reach into one that it writes: other CTAs, or other threads, still read it then.
struct Span { const void* p; int64_t words; };       // 32-bit words
bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || a.words <= 0 || b.words <= 0) return false;
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return x < y ? y - x < (uintptr_t)a.words * 4 : x - y < (uintptr_t)b.words * 4;
}
template <int N, int M>
bool any_overlap(const Span (&a)[N], const Span (&b)[M]) {
    for (const Span& x : a)
        for (const Span& y : b)
            if (overlap(x, y)) return true;
    return false;
}

}  // namespace

extern "C" int pkv_plan_step(const pkv_pages_t* pages, const int32_t* n_new_dev, const int32_t* parents_dev, const pkv_plan_t* plan,
                             void* stream) {
    int st = check_pages(pages);
    if (st) return st;
    if (!n_new_dev || !plan || !plan->cu_dev || !plan->ticket_dev || plan->capacity < 0) return PKV_ERR_INVALID;
    if (plan->capacity > 0x3fffffff) return PKV_ERR_UNSUPPORTED;
    // several CTAs read what the caller gives, and the tables, while the first already writes
    const int64_t cap = plan->capacity, B = pages->batch;
    const Span read[] = {{n_new_dev, B}, {parents_dev, cap}, {pages->page_table_dev, B * pages->max_pages}, {pages->seqlens_dev, B},
                         {pages->free_dev, (int64_t)pages->n_pages + 1}};
    const Span written[] = {{plan->cu_dev, B + 1}, {plan->seq_dev, cap}, {plan->positions_dev, cap}, {plan->slots_dev, cap}, {plan->mask_dev, 2 * cap},
                            {plan->ticket_dev, 1}, {plan->status_dev, 4}};
    if (any_overlap(read, written)) return PKV_ERR_INVALID;
    if (plan->capacity > 0 && (!plan->seq_dev || !plan->positions_dev || !plan->slots_dev || (parents_dev && !plan->mask_dev))) return PKV_ERR_INVALID;
    if (pages->batch == 0) return PKV_OK;
    PlanArgs A{*pages, *plan, n_new_dev, parents_dev};
    const int ctas = plan->capacity <= FILL ? 1 : (plan->capacity + FILL - 1) / FILL;
    PKV_CUDA_TRY(pkv_launch_chained(pkv_plan_step_kernel, dim3(ctas < 128 ? ctas : 128), dim3(NT), 0, (cudaStream_t)stream, A));
    return PKV_OK;
}

extern "C" int pkv_truncate(const pkv_pages_t* pages, const int32_t* lengths_dev, int32_t* status_dev, void* stream) {
    int st = check_pages(pages);
    if (st) return st;
    if (!lengths_dev) return PKV_ERR_INVALID;
    const Span read[] = {{lengths_dev, pages->batch}};
    const Span written[] = {{pages->page_table_dev, (int64_t)pages->batch * pages->max_pages}, {pages->seqlens_dev, pages->batch},
                            {pages->free_dev, (int64_t)pages->n_pages + 1}, {status_dev, 4}};
    if (any_overlap(read, written)) return PKV_ERR_INVALID;
    if (pages->batch == 0) return PKV_OK;
    PKV_CUDA_TRY(pkv_launch_chained(pkv_truncate_kernel, dim3(1), dim3(NT), 0, (cudaStream_t)stream, *pages, lengths_dev, status_dev));
    return PKV_OK;
}

extern "C" int pkv_keep_rows(const pkv_cache_t* const* layers, int32_t n_layers, const pkv_pages_t* pages, const int32_t* cu_dev,
                             int32_t capacity, const int32_t* keep_dev, const int32_t* n_keep_dev, int32_t* lengths_out_dev,
                             int32_t* status_dev, void* stream) {
    int st = check_pages(pages);
    if (st) return st;
    if (!layers || n_layers <= 0 || !cu_dev || (capacity > 0 && !keep_dev) || !n_keep_dev || capacity < 0) return PKV_ERR_INVALID;
    const int64_t B = pages->batch;
    const Span read[] = {{cu_dev, B + 1}, {keep_dev, capacity}, {n_keep_dev, B}, {pages->page_table_dev, B * pages->max_pages}, {pages->seqlens_dev, B}};
    const Span written[] = {{lengths_out_dev, B}, {status_dev, 4}};
    if (any_overlap(read, written)) return PKV_ERR_INVALID;
    for (int i = 0; i < n_layers; ++i) {
        const pkv_cache_t* c = layers[i];
        st = pkv_check_cache(c);
        if (st) return st;
        if (c->n_pages < pages->n_pages || c->n_kv <= 0 || c->head_dim <= 0) return PKV_ERR_INVALID;
        if (c->v_bits ? (c->head_dim != 128 || !c->vq_dev || (((uintptr_t)c->vq_dev) & 127u)) : (c->head_dim % 8 != 0 || (((uintptr_t)c->v_dev) & 15u)))
            return PKV_ERR_INVALID;
        for (int k = 0; k < i; ++k)                   // a pool given twice would be moved by two CTAs at once
            if (layers[k]->latent_dev == c->latent_dev || (c->v_dev && layers[k]->v_dev == c->v_dev) || (c->vq_dev && layers[k]->vq_dev == c->vq_dev))
                return PKV_ERR_INVALID;
    }
    if (pages->batch == 0) return PKV_OK;
    for (int i0 = 0; i0 < n_layers; i0 += MAX_LAYERS) {
        KeepArgs A = {};
        int units = 0, n = n_layers - i0 < MAX_LAYERS ? n_layers - i0 : MAX_LAYERS;
        for (int i = 0; i < n; ++i) {
            const pkv_cache_t* c = layers[i0 + i];
            uint8_t* v = (uint8_t*)(c->v_bits ? c->vq_dev : c->v_dev);
            A.layer[i] = KeepLayer{c->latent_dev, v, c->W, c->n_kv, c->head_dim, c->v_bits};
            const int u = keep_units(c->W, c->n_kv, c->head_dim, c->v_bits, v != nullptr);
            units = u > units ? u : units;
        }
        A.pg = *pages; A.cu = cu_dev; A.keep = keep_dev; A.n_keep = n_keep_dev; A.capacity = capacity;
        A.lengths_out = i0 == 0 ? lengths_out_dev : nullptr; A.status = status_dev;
        PKV_CUDA_TRY(pkv_launch_chained(pkv_keep_rows_kernel, dim3((units + KC - 1) / KC, pages->batch, n), dim3(KT), 0, (cudaStream_t)stream, A));
    }
    return PKV_OK;
}
