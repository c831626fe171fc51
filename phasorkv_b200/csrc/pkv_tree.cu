// Attention of a tree of drafted tokens over the paged latent cache.
//
//   S[i, h, t] = q'_{i,h} . c_t,   O[i, h] = softmax_t(S d^-1/2) V_{g(h)}   over t < base and t = base + j, bit j of mask_i
//
// with q' the absorbed query of drafted token i (conj(A) zq e^{i theta pos}; slow dims unrotated) and c_t the NVFP4 rows.
//
// The latent of a token serves all heads, so the rows of a score tile may be any mix of (kv head, drafted token, query
// head): a tile has 128 rows, `rph` for each of its G kv heads, and every CTA walks the pages of a sequence for one
// tile. Per page and tile:
//   S  [128 rows x 128 tokens]  = Q' . C^T     block-scaled NVFP4 tcgen05.mma, the four residual terms of the query added up
//                                              in tensor memory; a page is the B operand as it is stored
//   P  = 2^(S - m)              a thread per row and half page: maximum, sum and mask need no other lane
//   O^T[128 dims x rph] += V_g^T . P_g^T       bf16 tcgen05.mma, a kv head at a time, V as stored
// A tile of rows of several kv heads reads the latent page once for all of them, and one of 128 rows fills the M of the score MMA.
// With few drafted tokens a page's load, scores, softmax and P.V wait for one another with little slack between them: 131072 tokens, 8
// drafts: 70 us, 4.1 TB/s; 16 x 32768 tokens, 16 drafts: 266 us and 4.3 TB/s in short runs, 305 us and 3.8 TB/s in long ones, where the GPU
// draws its 1000 W and the clock falls to 1.54 GHz. With many drafts a page and tile takes 2450 cycles (8 x 8192 tokens, 64 drafts: 125 us in
// short runs, 138 in long ones at 1.76 GHz): 1536 of MMAs beside 1400 of exponentials and 1000 in which the warps hand over the page.
//
// Three launches: the operand (absorbed queries), the attention, the merge of what several CTAs did of one tile. (A last CTA that
// merges inside the attention launch waits for a counter and reads the others' partial results alone: slower than the third launch.)
#include "pkv_common.cuh"
#include "pkv_tcgen05.cuh"

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cudaTypedefs.h>
#include <cstring>

int pkv_check_layer(const pkv_layer_t* L);
int pkv_check_cache(const pkv_cache_t* c);

namespace {

using namespace pkv;

constexpr int DH = 128, ROWS = 128;                  // head dim; rows of a tile
constexpr int HALF = 64;                             // tokens per V stage: half a page of one kv head
constexpr int GROUP = 128;                           // threads of a softmax group: one per row of the tile; two groups, half a page each
constexpr int SOFT_WARPS = 2 * GROUP / 32;           // what they hand over is counted per warp: 32 arrivals at one word take turns
constexpr int MAX_G = 8;                             // kv heads of a tile (16 rows at least each)
constexpr float RESCALE_THRESHOLD = 8.0f;            // in base-2 logits
constexpr uint32_t WAIT_LIMIT = 1u << 19;            // probes of a bounded wait

// ------------------------------------------------------------------------------------------------ tiles and their pages
// How a sequence with n drafted tokens is cut into tiles: z = blk * groups + group covers `qpb` drafted tokens from blk * qpb on, kv
// heads group * G .. . Row r of a tile: kv head r / rph, drafted token (r % rph) / rep, query head (r % rph) % rep of the kv head.
struct Shape { int qpb, rph, G, groups, Z, cost; };
// What a page costs a tile: a score tile and its softmax, or, from two kv heads on, the values of the kv heads (in quarters of the
// former: 2500 cycles a page for one kv head, some 6000 for four).
constexpr int COST_ONE = 4, COST_MOST = 20;
constexpr int N_SM = 148;                            // CTAs of the attention launch: one per SM of a B200

struct Tiles {
    int rep, Z;                                      // query heads per kv head; most tiles of a sequence
    uint32_t rep_inv;                                // row / rep = row * rep_inv >> 16 for the rows of a tile
    int quantised;                                   // value pages hold codes
    uint32_t shape[PKV_TREE_MAX + 1];                // by drafted tokens: qpb - 1 | rph / 16 - 1 | G - 1 | groups - 1, 6 + 3 + 3 bits and the rest
    __device__ __forceinline__ Shape of(int n) const {
        const uint32_t w = shape[n];
        Shape t;
        t.qpb = (w & 63u) + 1; t.rph = ((w >> 6 & 7u) + 1) * 16; t.G = (w >> 9 & 7u) + 1; t.groups = (w >> 12) + 1;
        t.Z = t.groups * (n > t.qpb ? (n + t.qpb - 1) / t.qpb : 1);
        t.cost = quantised ? COST_ONE + t.G : max(COST_ONE, t.G * 5 / 2);
        return t;
    }
};

struct Batch {
    const int32_t *cu, *seqlens;
    int batch, max_pages, n_tokens, max_draft;
    // pages of sequence b, 0 when it has no drafted token or its numbers do not fit
    __device__ __forceinline__ int pages(int b, int& lo, int& n, int& T) const {
        lo = cu[b];
        n = cu[b + 1] - lo;
        T = seqlens[b];
        const bool ok = n > 0 && n <= max_draft && lo >= 0 && lo <= n_tokens - n && T >= n && T <= max_pages * PKV_PAGE_TOKENS;
        return ok ? (T + PKV_PAGE_TOKENS - 1) / PKV_PAGE_TOKENS : 0;
    }
};

// Work is a list: sequence by sequence, `passes` times over its pages. It is cut into stretches of U / gangs (the first U % gangs of
// them one longer), one per gang of CTAs; a page belongs to the stretch in which it begins, and the gang's CTA zi takes the tile
// pass * gang + zi of it. So every CTA has as much to do whatever the lengths are.
//   Every sequence has as many tiles (the usual step: as many drafts): a page counts 1, a gang has a CTA per tile (up to 16, then there are
//   passes), and the tiles of a sequence read a page at about the same time, from L2 all but the first.
//   Otherwise every CTA is a gang of its own, a sequence has a pass per tile, and a page counts what it costs the tile: no CTA idles
//   where a sequence has fewer tiles than another (24 ragged sequences of 0 .. 21 drafts, before later steps: 104 us; tiles of one
//   shape, by the most drafts, and gangs of them: 130 us).
struct List { int gang, gangs, U; };                 // gang: CTAs, or 0 for CTAs on their own
constexpr int LIST_WORDS = 5;

__device__ __forceinline__ int passes_of(const Shape& t, int gang) { return gang == 0 ? t.Z : (t.Z + gang - 1) / gang; }
__device__ __forceinline__ int cost_of(const Shape& t, int gang) { return gang == 0 ? t.cost : 1; }

// by all nt threads of a CTA; red: LIST_WORDS words per warp. last: pages and drafted tokens of the last sequence that the thread looked at
// (its only one, in batches of at most nt)
__device__ __forceinline__ List list_of(const Batch& B, const Tiles& X, int tid, int nt, int (*red)[LIST_WORDS], int2& last) {
    last = make_int2(0, 0);
    int v[LIST_WORDS] = {0, 0, 0, 1 << 30, 1};       // pages, pages x tiles x cost, most tiles, fewest tiles, highest cost
#pragma unroll 1
    for (int b = tid; b < B.batch; b += nt) {
        int lo, n, T;
        const int pages = B.pages(b, lo, n, T);
        last = make_int2(pages, n);
        if (pages == 0) continue;
        const Shape t = X.of(n);
        const int Z = t.Z;
        v[0] += pages; v[1] += pages * Z * t.cost;
        v[2] = max(v[2], Z); v[3] = min(v[3], Z); v[4] = max(v[4], t.cost);
    }
    v[0] = __reduce_add_sync(0xffffffffu, v[0]); v[1] = __reduce_add_sync(0xffffffffu, v[1]);
    v[2] = __reduce_max_sync(0xffffffffu, v[2]); v[3] = __reduce_min_sync(0xffffffffu, v[3]); v[4] = __reduce_max_sync(0xffffffffu, v[4]);
    if ((tid & 31) == 0)
#pragma unroll
        for (int i = 0; i < LIST_WORDS; ++i) red[tid >> 5][i] = v[i];
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < min(nt, B.batch + 31) / 32; ++w) {     // (the other warps have none)
        if (w == (tid >> 5)) continue;
        v[0] += red[w][0]; v[1] += red[w][1];
        v[2] = max(v[2], red[w][2]); v[3] = min(v[3], red[w][3]); v[4] = max(v[4], red[w][4]);
    }
    List y;
    const int passes = (v[2] + 15) >> 4;
    y.gang = v[2] == v[3] ? (v[2] + passes - 1) / passes : 0;
    y.gangs = y.gang ? N_SM / y.gang : N_SM;
    y.U = v[2] == v[3] ? v[0] * passes : v[1];
    // (a stretch that is not its tile's first or last has a page: none is shorter than the dearest page)
    y.gangs = min(y.gangs, y.gang ? y.U : max(y.U / v[4], min(y.U, 1)));
    return y;
}

struct Cut {
    int per, longer;                                 // pages of a stretch; how many have one more
    __device__ __forceinline__ Cut(int U, int gangs) : per(U / gangs), longer(U % gangs) {}
    __device__ __forceinline__ int start(int x) const { return x * per + min(x, longer); }
    __device__ __forceinline__ int of(int u) const {     // the stretch that page u of the list belongs to
        const int head = longer * (per + 1);
        return u < head ? u / (per + 1) : longer + (u - head) / per;
    }
};

struct Part {                                        // a stretch of pages of one tile
    int b, z, p_lo, p_hi, pages, lo, n, T;
    Shape t;
};

struct Walk {
    int b, pass, p, at, end, gang;                   // at: place on the list of the (sequence, pass); end: of the stretch
    __device__ __forceinline__ bool next(const Batch& B, const Tiles& X, int zi, Part& s) {
        while (at < end && b < B.batch) {
            s.pages = B.pages(b, s.lo, s.n, s.T);
            if (s.pages == 0) { ++b; continue; }
            s.t = X.of(s.n);
            const int cost = cost_of(s.t, gang), here = end - at;
            s.b = b; s.z = gang ? pass * gang + zi : pass; s.p_lo = p; s.p_hi = min(s.pages, (here + cost - 1) / cost);
            at = here > s.pages * cost ? at + s.pages * cost : end;
            p = 0;
            if (++pass == passes_of(s.t, gang)) { pass = 0; ++b; }
            if (s.p_lo < s.p_hi && s.z < s.t.Z) return true;         // else: this CTA has no tile in this pass
        }
        return false;
    }
};

// ------------------------------------------------------------------------------------------------ operand
// two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*reinterpret_cast<unsigned long long*>(&d)) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&d)) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&d)) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// One residual term of 16 columns: E4M3 scale (in units of the row's `second`) and E2M1 codes; res becomes what is left. The
// next term is formed from what was stored, so any rounding will do: hardware conversions and an approximate reciprocal.
__device__ __forceinline__ uint2 residual_term(float (&res)[16], float second, float inv_second, uint8_t& sb, bool more) {
    float am = fabsf(res[0]);
#pragma unroll
    for (int i = 1; i < 15; i += 2) am = max3(am, fabsf(res[i]), fabsf(res[i + 1]));
    am = fmaxf(am, fabsf(res[15]));
    sb = pkv_float_to_e4m3(am * (1.0f / 6.0f) * inv_second);
    const float scale = pkv_e4m3_to_float(sb) * second;
    float inv;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    if (sb == 0) inv = 0.0f;
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = mul2(make_float2(res[8 * h + 2 * i], res[8 * h + 2 * i + 1]), make_float2(inv, inv));
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(w[h]) : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
    }
    if (more) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2_raw p = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(w[h] >> (8 * i)), __NV_E2M1);
                const float2 f = fma2(__half22float2(__half2(p)), make_float2(-scale, -scale), make_float2(res[8 * h + 2 * i], res[8 * h + 2 * i + 1]));
                res[8 * h + 2 * i] = f.x;
                res[8 * h + 2 * i + 1] = f.y;
            }
        }
    }
    return make_uint2(w[0], w[1]);
}

// Tile operand of a (sequence, tile): four residual terms, each a 128-row tile laid out like a cache page (swizzled codes,
// then the block scales), and 128 fp32 row scales.
__host__ __device__ constexpr int page_bytes(int WP) { return PKV_PAGE_TOKENS * WP / 2 + WP / 64 * 512; }
__host__ __device__ constexpr int blob_bytes(int WP) { return PKV_QUERY_TERMS * page_bytes(WP) + ROWS * 4; }

struct AbsorbArgs {
    pkv_layer_t L;
    Batch B;
    Tiles X;
    const void* q;
    int q_bf16;
    const int32_t* positions;
    uint8_t* blobs;
    int32_t* first_page;
    int32_t* status;
};

constexpr int AR = 16;                               // rows per CTA

// CTA (16 rows of a tile, tile, sequence): a thread per column for the absorbed rows, then a thread per row and block of 16 columns for
// the terms. Rows that no drafted token has are not written: a row of garbage only reaches its own column of the result, which nobody
// reads. Latency with few drafts (6 us: lengths, queries and factors from cold memory), instruction issue with many (16384 rows of 256
// columns: 15 us, 18 with the loads one after the other and the terms formed a value at a time).
// The launch behind it is let go at once although its pages then compete with this one's loads: 74 us against 75 when the queries have
// arrived and 78 at the end (131072 tokens, 8 drafts).
template <int WP>
__global__ void __launch_bounds__(AR * WP / 16) pkv_tree_absorb_kernel(const AbsorbArgs A) {
    constexpr int NB = WP / 16, NT = AR * NB, RB = WP / 2;
    static_assert(NT == WP, "a thread per column");
    // raw queries and phasors first, later (in the same place) the absorbed rows
    // (a block of 16 absorbed columns takes 20 words: a thread reads a block, and the blocks of a row then start in different banks)
    constexpr int PITCH = NB * 20 + 4, FIRST = AR * DH * 4 + AR * DH / 2 * 8, THEN = AR * PITCH * 4;
    __shared__ __align__(16) uint8_t both[FIRST > THEN ? FIRST : THEN];
    __shared__ float2 zq[AR][DH / 2];
    __shared__ int sums[NT / 32][LIST_WORDS];
    float (*raw)[DH] = reinterpret_cast<float (*)[DH]>(both);
    float2 (*ph)[DH / 2] = reinterpret_cast<float2 (*)[DH / 2]>(both + AR * DH * 4);
    float (*qa)[PITCH] = reinterpret_cast<float (*)[PITCH]>(both);
    const pkv_layer_t& L = A.L;
    const int tid = threadIdx.x, z = blockIdx.y, b = blockIdx.z, r0 = blockIdx.x * AR;
    pkv_grid_wait();                                 // everything before this launch is done ..
    pkv_grid_launch_dependents();                    // .. so the attention behind it may stream pages while this one still runs
    // One more CTA per sequence, for the merge: the sequence's place on the list; the last sequence's: the list itself.
    if (blockIdx.x == ROWS / AR) {
        if (z != 0) return;
        int2 last;
        const List y = list_of(A.B, A.X, tid, NT, sums, last);
        int before = 0;
#pragma unroll 1
        for (int i = tid; i < b; i += NT) {
            int lo, n, T;
            const int pages = A.B.pages(i, lo, n, T);
            if (pages) { const Shape t = A.X.of(n); before += pages * passes_of(t, y.gang) * cost_of(t, y.gang); }
        }
        before = __reduce_add_sync(0xffffffffu, before);
        __syncthreads();
        if ((tid & 31) == 0) sums[tid >> 5][0] = before;
        __syncthreads();
        if (tid == 0) {
            before = 0;
#pragma unroll 1
            for (int w = 0; w < NT / 32; ++w) before += sums[w][0];
            A.first_page[b] = before;
            if (b == A.B.batch - 1) { A.first_page[b + 1] = y.U; A.first_page[b + 2] = y.gang; A.first_page[b + 3] = y.gangs; }
        }
        return;
    }
    int lo, n, T;
    const int pages = A.B.pages(b, lo, n, T);
    if (pages == 0) {
        if (n != 0 && tid == 0 && blockIdx.x == 0 && z == 0) pkv_report(A.status, 4, b);
        return;
    }
    const Shape t = A.X.of(n);
    if (z >= t.Z) return;
    const int rep = A.X.rep, blk = z / t.groups, first = blk * t.qpb, nq = min(t.qpb, n - first);
    const int g = z % t.groups * t.G + r0 / t.rph, rr0 = r0 % t.rph;      // rph is a multiple of 16: one kv head per CTA
    const int rows = min(AR, nq * rep - rr0);
    if (nq <= 0 || r0 / t.rph >= t.G || g >= L.n_kv || rows <= 0) return;
    // this CTA's rows belong to the drafted tokens q_lo .. q_hi
    auto token = [&](int row) { return (int)(row * A.X.rep_inv >> 16); };
    const int q_lo = token(rr0), q_hi = token(rr0 + rows - 1);
    // the factors of this thread's column, used for all rows
    const int R = L.R, W = 2 * R + L.R_s, c = tid;
    int f = 0;
    float ar = 0.0f, ai = 0.0f, tier = 1.0f;
    if (c < 2 * R) {
        const int k = c < R ? c : c - R;
        f = L.freq_dev[k];
        ar = L.A_re_dev[g * R + k];
        ai = L.A_im_dev[g * R + k];
    }
    // tiers: the cache's block is in units of its own scale while the attention applies the layer's one
    if (L.second_blocks_dev && c < W) tier = L.second_blocks_dev[c >> 4] / L.second;
    constexpr int QL = AR * (DH / 4) / NT;               // four dims at a time; all loads of a thread in flight
    float4 qv[QL];
#pragma unroll
    for (int i = 0; i < QL; ++i) {
        const int k = tid + i * NT, r = k / (DH / 4), d = k % (DH / 4) * 4, rr = rr0 + r, tk = token(rr);
        const size_t o = ((size_t)(lo + first + tk) * L.n_q + g * rep + rr - tk * rep) * DH + d;
        if (r >= rows) continue;
        if (A.q_bf16) {
            const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*)A.q + o);
            qv[i] = make_float4(pkv_bf16_bits_to_float(u.x & 0xffffu), pkv_bf16_bits_to_float(u.x >> 16), pkv_bf16_bits_to_float(u.y & 0xffffu),
                                pkv_bf16_bits_to_float(u.y >> 16));
        } else {
            qv[i] = *reinterpret_cast<const float4*>((const float*)A.q + o);
        }
    }
    // Phasors: the angle as a number of turns in 64 bits, of which only the fraction counts; that is exact enough in 32 bits
    // (2^-25 of a turn) and needs no long range reduction (the operand's own residual is 7e-5).
#pragma unroll 1
    for (int k = tid; k < (q_hi - q_lo + 1) * (DH / 2); k += NT) {
        const int j = k % (DH / 2);
        const double turns = (double)A.positions[lo + first + q_lo + k / (DH / 2)] * L.inv_freq_dev[j] * 0.15915494309189533577;
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        ph[k / (DH / 2)][j] = make_float2(L.attn_scale * cs, L.attn_scale * sn);
    }
#pragma unroll
    for (int i = 0; i < QL; ++i) {
        const int k = tid + i * NT;
        if (k / (DH / 4) < rows) *reinterpret_cast<float4*>(&raw[k / (DH / 4)][k % (DH / 4) * 4]) = qv[i];
    }
    __syncthreads();
#pragma unroll 2
    for (int k = tid; k < rows * (DH / 2); k += NT) {
        const int r = k / (DH / 2), j = k % (DH / 2);
        const float2 p = ph[token(rr0 + r) - q_lo][j];
        const float x = raw[r][j], y = raw[r][j + DH / 2];
        zq[r][j] = make_float2(x * p.x - y * p.y, x * p.y + y * p.x);
    }
    __syncthreads();
    // absorbed rows: a column per thread
    float acc[AR] = {};
    if (c >= 2 * R && c < W) {                       // slow dims: the raw query; a factor serves all rows
#pragma unroll 4
        for (int s = 0; s < 2 * L.n_slow; ++s) {
            const int d = s < L.n_slow ? L.slow_dev[s] : L.slow_dev[s - L.n_slow] + DH / 2;
            const float a = L.A_s_dev[((size_t)g * 2 * L.n_slow + s) * L.R_s + c - 2 * R];
#pragma unroll
            for (int r = 0; r < AR; ++r) acc[r] = fmaf(raw[r][d], a, acc[r]);
        }
    }
    __syncthreads();                                 // the raw queries are done with
    // conj(A) zq: (ar x + ai y, ar y - ai x), of which the column has one; padding: 0
    const float ax = c < R ? ar : -ai, ay = c < R ? ai : ar;
    float* column = &qa[0][(c >> 4) * 20 + (c & 15)];
#pragma unroll
    for (int r = 0; r < AR; ++r) {
        if (c < 2 * R) {
            const float2 w = zq[r][f];
            acc[r] = fmaf(ax, w.x, ay * w.y);
        }
        column[r * PITCH] = acc[r] * tier;
    }
    __syncthreads();
    const int r = tid / NB, j = tid % NB;            // from here on: a 16-column block of a row per thread
    const bool live = r < rows;
    float res[16];
    float2 none = make_float2(0.0f, 0.0f);           // NaN as soon as a value is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(&res[4 * i]) = *reinterpret_cast<const float4*>(&qa[r][j * 20 + 4 * i]);
    float am = fmaxf(fabsf(res[0]), fabsf(res[15]));
#pragma unroll
    for (int i = 0; i < 16; i += 2) none = fma2(make_float2(res[i], res[i + 1]), make_float2(0.0f, 0.0f), none);
#pragma unroll
    for (int i = 1; i < 15; i += 2) am = max3(am, fabsf(res[i]), fabsf(res[i + 1]));
#pragma unroll
    for (int o = NB / 2; o; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
    const uint32_t bad = __ballot_sync(0xffffffffu, !(none.x + none.y == 0.0f));
    const bool fine = (bad >> ((tid & 31) / NB * NB) & ((1u << NB) - 1)) == 0;
    if (!live) return;
    const float second = fmaxf(am, 1e-30f) * (1.0f / (448.0f * 6.0f)), inv = __frcp_rn(second);
    uint8_t* blob = A.blobs + ((size_t)b * A.X.Z + z) * blob_bytes(WP);
    const uint32_t row = r0 + r;
#pragma unroll 1
    for (int t = 0; t < PKV_QUERY_TERMS; ++t) {
        uint8_t sb;
        const uint2 packed = residual_term(res, second, inv, sb, t + 1 < PKV_QUERY_TERMS);
        uint8_t* tile = blob + t * page_bytes(WP);
        *reinterpret_cast<uint2*>(tile + pkv_code_offset(row, j * 8, RB)) = packed;
        tile[PKV_PAGE_TOKENS * RB + pkv_scale_offset(row, j)] = sb;
    }
    // a query that is not finite makes its whole row NaN
    if (j == 0) reinterpret_cast<float*>(blob + PKV_QUERY_TERMS * page_bytes(WP))[row] = fine ? second : __int_as_float(0x7fc00000);
}

// ------------------------------------------------------------------------------------------------ attention
// tensor memory columns
constexpr uint32_t TM_S = 0;          // 2 x 128: scores of a page, rows x tokens
constexpr uint32_t TM_O = 256;        // 128: O^T, dims x rows
constexpr uint32_t TM_SFA = 384;      // 4 per (term, K step): scales of the query
constexpr uint32_t TM_SFB = 448;      // 2 x 16: scales of the page
constexpr uint32_t TM_COLS = 512;

// MANY: tiles of two kv heads or more, of bf16 values. Of wide rows, their values are most of what a page brings, and the page after next can
// wait: one latent page and four stages of values instead of two and three (16 x 16384 tokens, 6 drafts, 4 kv heads per tile: 140 -> 123 us;
// 32 drafts of one kv head per tile: 134 -> 150 us). The exponentials differ too, see there.
template <int WP, bool VQ, bool MANY>
struct Cfg {
    static constexpr int RB = WP / 2, KB = WP / 64, PAGE = page_bytes(WP), CODES = PKV_PAGE_TOKENS * RB;
    static constexpr int NK = WP == 256 ? (MANY ? 1 : 2) : 4;                                  // latent pages in flight
    // V operand stages (64 tokens of a kv head, bf16) and, of quantised V, raw stages: what is left of the shared memory
    static constexpr int NV = VQ ? (WP == 256 ? 2 : 3) : (WP == 256 ? (MANY ? 4 : 3) : 5);
    static constexpr int NR = VQ ? (WP == 256 ? 3 : 8) : 0;
    static constexpr int V_BYTES = HALF * DH * 2, RAW_BYTES = HALF * DH / 2, P_BYTES = ROWS * PKV_PAGE_TOKENS * 2;
    static constexpr int SC_BYTES = MAX_G * PKV_PAGE_TOKENS * 2;                  // token scales of a page
    static constexpr int Q_OFF = 0;
    static constexpr int K_OFF = (blob_bytes(WP) + 1023) / 1024 * 1024;
    static constexpr int V_OFF = K_OFF + NK * PAGE;
    static constexpr int P_OFF = V_OFF + NV * V_BYTES;
    static constexpr int R_OFF = P_OFF + 2 * P_BYTES;                             // weights: a buffer per softmax group
    static constexpr int SC_OFF = R_OFF + NR * RAW_BYTES;
    static constexpr int X_OFF = SC_OFF + (VQ ? 2 * SC_BYTES : 0);
    static constexpr int SMEM = X_OFF + 6144;
    static constexpr int NTHREADS = VQ ? 512 : 384;
    static constexpr uint64_t SWZ = RB == 128 ? SWZ_128B : SWZ_64B;
    static_assert(!MANY || !VQ, "of bf16 values alone");
    static_assert(SMEM <= 232448 && V_OFF % 1024 == 0 && P_OFF % 1024 == 0, "shared memory of a CTA");
};

struct Shared {                       // at X_OFF
    uint64_t q_full[PKV_QUERY_TERMS], q_empty, o_empty;
    uint64_t p_full[2], pv_done[2];
    uint64_t k_full[4], k_empty[4], v_full[7], v_empty[7], v_clean[7], s_full[2], s_empty[2];
    uint64_t r_full[8], r_empty[8], sc_full[2], sc_empty[2], drained[2];
    uint32_t tmem_base;
    volatile int abort_flag;
    Walk start;
    alignas(16) float row_f[2][ROWS]; // rescale factors; at the end, per group: 1 / sum
    float row_l[2][ROWS];             // per group: a page's maxima where a reference moves; sums at the end
    uint32_t bad[3][MAX_G][2];        // [stretch % 3]: drafted tokens whose value row of a kv head is not finite
    int scan[16], red[16][LIST_WORDS];
    alignas(16) int row_o[2][ROWS];   // per group: where a row's result goes, or -1
};
static_assert(sizeof(Shared) <= 6144, "behind the stages");

__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, Shared* X, int32_t* status, int where) {
    for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && X->abort_flag) return false;
    }
    X->abort_flag = 1;
    pkv_report(status, 1, where);
    return false;
}
// bounded; false when it gave up, or another role did (out of line: it is in many places, and the code has to stay small)
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, Shared* X, int32_t* status, int where) {
    return mbar_try_wait(bar, parity) || wait_longer(bar, parity, X, status, where);
}

// a value that all lanes hold, as one the compiler knows to be uniform (a warp reduction ends in a uniform register)
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// the 256 softmax threads meet (named barrier 3) and learn whether the predicate held in any of them
__device__ __forceinline__ bool softmax_any(bool pred) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 3, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(pred ? 1 : 0) : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 3, 256;" ::: "memory"); }
// the 128 threads of a group (named barrier 1 or 2)
__device__ __forceinline__ void group_sync(int group) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + group) : "memory"); }

// one arrival for the warp, behind everything its lanes did
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ float ex2_fast(float x) {     // 2 ulp, results below 2^-126 become 0: a weight needs no more
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The same for two numbers without the exponential unit, which the softmax keeps busy: n = rint(x), and 2^(x - n) by the cubic of least
// relative error on -1/2 .. 1/2 (7.5e-5, a twenty-sixth of half a bf16 step; coefficients by linear programming on 4001 points). NaN stays NaN; below 2^-126 (-infinity too): 0.
__device__ __forceinline__ float2 ex2_cubic(float2 x) {
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x.x) : "f"(x.x), "f"(-127.0f));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x.y) : "f"(x.y), "f"(-127.0f));
    const float2 t = add2(x, make_float2(12582912.0f, 12582912.0f)), n = add2(t, make_float2(-12582912.0f, -12582912.0f));      // 1.5 x 2^23
    const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
    float2 y = fma2(f, make_float2(0.055171670f, 0.055171670f), make_float2(0.242611125f, 0.242611125f));
    y = fma2(f, y, make_float2(0.693260985f, 0.693260985f));
    y = fma2(f, y, make_float2(0.999928073f, 0.999928073f));
    return mul2(y, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

struct AttnArgs {
    Batch B;
    Tiles X;
    const int32_t* page_table;
    const int64_t* mask;
    const uint8_t* blobs;
    const uint8_t* vq;
    int n_pages, n_kv, n_q;
    float col_scale;                  // tensor scale of the latent x log2(e) / sqrt(d)
    float* part_o;                    // [2 per CTA][128 rows][128 dims]
    float2* part_ml;                  // [2 per CTA][128 rows]
    const int32_t* first_page;        // [batch + 3]: each sequence's first page on the list; all pages, CTAs per gang, gangs
    __nv_bfloat16* out;
    int32_t* status;
};

template <int WP, bool VQ, bool MANY>
__global__ void __launch_bounds__(Cfg<WP, VQ, MANY>::NTHREADS, 1) pkv_tree_attn_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                                 const __grid_constant__ CUtensorMap qmap,
                                                                                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnArgs A) {
    using C = Cfg<WP, VQ, MANY>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared* X = reinterpret_cast<Shared*>(smem + C::X_OFF);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Tiles& tl = A.X;
    pkv_grid_launch_dependents();

    // ---- barriers, tensor memory, and where on the list of pages this CTA starts. Page table, lengths, masks and pages are
    // final: the operand launch in front of this one has started, so everything before that is done.
    // (Code that runs once per CTA costs what its bytes take to fetch: it is kept short, loops are left rolled.)
    if (warp == 0) {                                 // lane i takes entry i of every array
        if (lane == 0) {
            mbar_init(&X->q_empty, SOFT_WARPS + 1); mbar_init(&X->o_empty, SOFT_WARPS);
            X->abort_flag = 0;
            X->start = Walk{0, 0, 0, 0, 0, 0};
        }
        if (lane < PKV_QUERY_TERMS) mbar_init(&X->q_full[lane], 1);
        if (lane < 2) {
            mbar_init(&X->p_full[lane], SOFT_WARPS); mbar_init(&X->pv_done[lane], 1); mbar_init(&X->s_full[lane], 1); mbar_init(&X->s_empty[lane], SOFT_WARPS);
            mbar_init(&X->sc_full[lane], 1); mbar_init(&X->sc_empty[lane], SOFT_WARPS); mbar_init(&X->drained[lane], 1);
        }
        if (lane < C::NK) { mbar_init(&X->k_full[lane], 1); mbar_init(&X->k_empty[lane], 1); }
        if (lane < C::NV) { mbar_init(&X->v_full[lane], VQ ? 4 : 1); mbar_init(&X->v_empty[lane], 1); mbar_init(&X->v_clean[lane], SOFT_WARPS); }
        if (lane < C::NR) { mbar_init(&X->r_full[lane], 1); mbar_init(&X->r_empty[lane], 4); }
        fence_barrier_init();
    }
    if (tid < 3 * MAX_G * 2) (&X->bad[0][0][0])[tid] = 0u;
    if (warp == 3) tmem_alloc(&X->tmem_base, TM_COLS);
    tc_fence_before_sync();
    {
        int2 last;
        const List y = list_of(A.B, tl, tid, C::NTHREADS, X->red, last);
        const int per = (A.B.batch + C::NTHREADS - 1) / C::NTHREADS, b_lo = min(tid * per, A.B.batch), b_hi = min(b_lo + per, A.B.batch);
        int mine = 0, lo, n, T;
        auto pages_of = [&](int b) { if (per == 1) { n = last.y; return last.x; } return A.B.pages(b, lo, n, T); };
#pragma unroll 1
        for (int b = b_lo; b < b_hi; ++b) {
            const int pages = pages_of(b);
            if (pages) { const Shape t = tl.of(n); mine += pages * passes_of(t, y.gang) * cost_of(t, y.gang); }
        }
        int before = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) X->scan[warp] = before;
        __syncthreads();
        before -= mine;
#pragma unroll 1
        for (int w = 0; w < min(warp, (A.B.batch + 31) / 32); ++w) before += X->scan[w];
        const int gang = y.gang ? blockIdx.x / y.gang : blockIdx.x;
        if (gang < y.gangs) {
            const Cut cut(y.U, y.gangs);
            const int u0 = cut.start(gang);
            if (before <= u0 && u0 < before + mine) {
                int u = u0 - before;
#pragma unroll 1
                for (int b = b_lo; b < b_hi; ++b) {
                    const int pages = pages_of(b);
                    if (pages == 0) continue;
                    const Shape t = tl.of(n);
                    const int cost = cost_of(t, y.gang), block = pages * cost, units = block * passes_of(t, y.gang);
                    if (u < units) {
                        X->start = Walk{b, u / block, (u % block + cost - 1) / cost, u0 - u % block, cut.start(gang + 1), y.gang};
                        break;
                    }
                    u -= units;
                }
            }
        }
    }
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tb = X->tmem_base, sbase = smem_u32(smem);
    Walk walk = X->start;
    const int zi = walk.gang ? blockIdx.x % walk.gang : 0;
    Part s;
    auto drain = [&](bool leader, int i) {           // given up: the MMAs in flight end before the tensor memory goes back
        if (!X->abort_flag) return;
        if (leader) tc_commit(&X->drained[i]);
        mbar_wait(&X->drained[i], 0, 1u << 16);
    };
    auto heads = [&](const Part& p) { return min(p.t.G, A.n_kv - p.z % p.t.groups * p.t.G); };      // kv heads of the tile

    if (warp == 0) {
        // ================================================================== latent pages and query operand
        if (lane == 0) {
            tma_prefetch_desc(&kmap); tma_prefetch_desc(&qmap);
            int k = 0, seg = 0, n_sc = 0;
            bool ok = true, waited = false;
            while (ok && walk.next(A.B, tl, zi, s)) {
                for (int p = s.p_lo; p < s.p_hi && ok; ++p, ++k) {
                    const int st = k % C::NK, page = A.page_table[(size_t)s.b * A.B.max_pages + p];
                    if (page < 0 || page >= A.n_pages) {               // never dereferenced
                        X->abort_flag = 1;
                        pkv_report(A.status, 2, p);
                        ok = false;
                        break;
                    }
                    if (k >= C::NK) ok = wait_or_abort(&X->k_empty[st], (k / C::NK - 1) & 1, X, A.status, 10);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&X->k_full[st], C::PAGE);
                    tma_load_2d(smem + C::K_OFF + st * C::PAGE, &kmap, 0, page * (C::PAGE / 128), &X->k_full[st]);
                    if (p == s.p_lo) {                                  // the tile's operand, behind its first page
                        if (seg > 0) ok = wait_or_abort(&X->q_empty, (seg - 1) & 1, X, A.status, 11);
                        if (!ok) { ++k; break; }
                        if (!waited) { pkv_grid_wait(); waited = true; }
                        asm volatile("fence.proxy.async;" ::: "memory");   // written by ordinary stores, read by the copy engine
                        const long blob = (long)s.b * tl.Z + s.z;
                        for (int t = 0; t < PKV_QUERY_TERMS; ++t) {    // (the scores of a term begin when it is there)
                            const bool last = t + 1 == PKV_QUERY_TERMS;
                            mbar_arrive_expect_tx(&X->q_full[t], C::PAGE + (last ? ROWS * 4 : 0));
                            tma_load_2d(smem + C::Q_OFF + t * C::PAGE, &qmap, 0, (int)(blob * (blob_bytes(WP) / 128) + t * (C::PAGE / 128)), &X->q_full[t]);
                            if (last) bulk_g2s(smem + C::Q_OFF + PKV_QUERY_TERMS * C::PAGE, A.blobs + blob * blob_bytes(WP) + PKV_QUERY_TERMS * C::PAGE, ROWS * 4, &X->q_full[t]);
                        }
                        ++seg;
                    }
                    if constexpr (VQ) {
                        // The token scales of the page's kv heads. (Here and not with the tiles, behind which they would come when the
                        // ring of tiles has moved on, a whole page late: 16 x 16384 tokens, 12 drafts took 217 us instead of 190, now 163.)
                        const int g0 = s.z % s.t.groups * s.t.G, bytes = heads(s) * PKV_PAGE_TOKENS * 2;
                        if (k >= 2) ok = wait_or_abort(&X->sc_empty[k & 1], ((k >> 1) - 1) & 1, X, A.status, 22);
                        if (!ok) { ++k; break; }
                        mbar_arrive_expect_tx(&X->sc_full[k & 1], bytes);
                        bulk_g2s(smem + C::SC_OFF + (k & 1) * C::SC_BYTES,
                                 A.vq + (size_t)page * A.n_kv * PKV_VQ_TILE_BYTES + (size_t)A.n_kv * 8192 + g0 * 256, bytes, &X->sc_full[k & 1]);
                        n_sc = k + 1;
                    }
                }
            }
            if (!waited) pkv_grid_wait();
            if (X->abort_flag) {                                        // copies in flight land before anyone leaves
                for (int t = 0; t < PKV_QUERY_TERMS && seg > 0; ++t) mbar_wait(&X->q_full[t], (seg - 1) & 1, 1u << 16);
                for (int j = max(0, k - C::NK); j < k; ++j) mbar_wait(&X->k_full[j % C::NK], (j / C::NK) & 1, 1u << 16);
                for (int j = max(0, n_sc - 2); j < n_sc; ++j) mbar_wait(&X->sc_full[j & 1], (j >> 1) & 1, 1u << 16);
            }
        }
    } else if (warp == 1) {
        // ================================================================== values
        if (lane == 0) {
            tma_prefetch_desc(&vmap);
            int k = 0;
            bool ok = true;
            while (ok && walk.next(A.B, tl, zi, s)) {
                const int g0 = s.z % s.t.groups * s.t.G, ng = heads(s);
                for (int p = s.p_lo; p < s.p_hi && ok; ++p) {
                    const int page = A.page_table[(size_t)s.b * A.B.max_pages + p];
                    if (page < 0 || page >= A.n_pages) { ok = false; break; }      // (reported by warp 0)
                    for (int j = 0; j < 2 * ng && ok; ++j, ++k) {
                        if constexpr (VQ) {
                            const int st = k % (C::NR ? C::NR : 1);
                            if (k >= C::NR) ok = wait_or_abort(&X->r_empty[st], (k / C::NR - 1) & 1, X, A.status, 21);
                            if (!ok) break;
                            mbar_arrive_expect_tx(&X->r_full[st], C::RAW_BYTES);
                            tma_load_2d(smem + C::R_OFF + st * C::RAW_BYTES, &vmap, 0, page * A.n_kv * (PKV_VQ_TILE_BYTES / 128) + (g0 + (j >> 1)) * 64 + (j & 1) * 32,
                                        &X->r_full[st]);
                        } else {
                            const int st = k % C::NV, y = (page * A.n_kv + g0 + (j >> 1)) * PKV_PAGE_TOKENS + (j & 1) * HALF;
                            if (k >= C::NV) ok = wait_or_abort(&X->v_empty[st], (k / C::NV - 1) & 1, X, A.status, 20);
                            if (!ok) break;
                            uint8_t* dst = smem + C::V_OFF + st * C::V_BYTES;
                            mbar_arrive_expect_tx(&X->v_full[st], C::V_BYTES);
                            tma_load_2d(dst, &vmap, 0, y, &X->v_full[st]);
                            tma_load_2d(dst + C::V_BYTES / 2, &vmap, 64, y, &X->v_full[st]);
                        }
                    }
                }
            }
            if (X->abort_flag) {                                        // copies in flight land before anyone leaves
                if constexpr (VQ) {
                    for (int j = max(0, k - C::NR); j < k; ++j) mbar_wait(&X->r_full[j % (C::NR ? C::NR : 1)], (j / (C::NR ? C::NR : 1)) & 1, 1u << 16);
                } else {
                    for (int j = max(0, k - C::NV); j < k; ++j) mbar_wait(&X->v_full[j % C::NV], (j / C::NV) & 1, 1u << 16);
                }
            }
        }
    } else if (warp == 2) {
        // ================================================================== score MMAs, issued by one elected lane
        // The whole warp runs the loop, so that every operand of an MMA is warp-uniform: in a branch of one lane the compiler
        // moves each descriptor through vector registers, and the issue (about 130 cycles an MMA) takes longer than the MMA.
        // Scores and P.V are issued by a warp each: one that waits for values must not hold up the next page's scores.
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = idesc_nvfp4(ROWS, PKV_PAGE_TOKENS);
        const uint64_t q_desc = smem_desc(sbase + C::Q_OFF, 0, 8 * C::RB, C::SWZ);
        int k = 0, seg = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
            ok = __all_sync(0xffffffffu, ok && wait_or_abort(bar, parity, X, A.status, where));
        };
        while (ok && walk.next(A.B, tl, zi, s)) {
            const int p_lo = uniform(s.p_lo), p_hi = uniform(s.p_hi);
            for (int p = p_lo; p < p_hi; ++p, ++k) {
                const int st = k % C::NK, sb = k & 1;
                wait(&X->k_full[st], (k / C::NK) & 1, 33);
                if (k >= 2) wait(&X->s_empty[sb], ((k >> 1) - 1) & 1, 34);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t ka = sbase + C::K_OFF + st * C::PAGE, sfb = tb + TM_SFB + 16 * sb;
                const uint64_t k_desc = smem_desc(ka, 0, 8 * C::RB, C::SWZ), sf_desc = smem_desc(ka + C::CODES, 0, 128, SWZ_NONE);
                if (leader)
#pragma unroll
                    for (int c = 0; c < C::KB; ++c) tmem_cp_32x128b_warpx4(sfb + 4 * c, sf_desc + (uint64_t)(c * 512 / 16));
#pragma unroll 1
                for (int t = 0; t < PKV_QUERY_TERMS; ++t) {
                    if (p == p_lo) {                     // the tile's operand arrives term by term
                        wait(&X->q_full[t], seg & 1, 30);
                        if (!ok) break;
                        tc_fence_after_sync();
                        if (leader)
#pragma unroll
                            for (int c = 0; c < C::KB; ++c)
                                tmem_cp_32x128b_warpx4(tb + TM_SFA + (t * C::KB + c) * 4, smem_desc(sbase + C::Q_OFF + t * C::PAGE + C::CODES + c * 512, 0, 128, SWZ_NONE));
                        __syncwarp();
                    }
                    if (leader)
#pragma unroll
                        for (int c = 0; c < C::KB; ++c)
                            mma_nvfp4(tb + TM_S + 128 * sb, q_desc + (uint64_t)((t * C::PAGE + c * 32) / 16), k_desc + (uint64_t)(c * 32 / 16), idesc_s,
                                      tb + TM_SFA + (t * C::KB + c) * 4, sfb + 4 * c, t != 0 || c != 0);
                }
                if (!ok) break;
                if (leader) {
                    tc_commit(&X->k_empty[st]);
                    tc_commit(&X->s_full[sb]);
                    if (p + 1 == p_hi) tc_commit(&X->q_empty);
                }
                __syncwarp();
            }
            ++seg;
        }
        drain(leader, 0);
    } else if (warp == 3) {
        // ================================================================== P.V MMAs: O^T += V^T P^T
        const bool leader = elect_one();
        const uint64_t p_desc = smem_desc(sbase + C::P_OFF, 0, 1024, SWZ_128B);
        int k = 0, kv = 0, seg = 0;
        uint32_t cleaned = 0;                          // phase bit of every stage's v_clean
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
            ok = __all_sync(0xffffffffu, ok && wait_or_abort(bar, parity, X, A.status, where));
        };
        while (ok && walk.next(A.B, tl, zi, s)) {
            const int ng = uniform(heads(s)), base = uniform(s.T - s.n), rph = uniform(s.t.rph);
            const uint32_t idesc_o = idesc_bf16(DH, rph, true, false);
            const int p_lo = uniform(s.p_lo), p_hi = uniform(s.p_hi);
            for (int p = p_lo; p < p_hi && ok; ++p, ++k) {
                wait(&X->p_full[k & 1], (k >> 1) & 1, 31);
                if (p == p_lo && seg > 0) wait(&X->o_empty, (seg - 1) & 1, 35);
                const bool tail = !VQ && base < (p + 1) * PKV_PAGE_TOKENS;     // rows that are no cached tokens: looked over first
                for (int j = 0; j < 2 * ng && ok; ++j, ++kv) {
                    const int st = kv % C::NV, g = j >> 1, h = j & 1;
                    wait(&X->v_full[st], (kv / C::NV) & 1, 32);
                    if (tail) {
                        wait(&X->v_clean[st], cleaned >> st & 1, 36);
                        cleaned ^= 1u << st;
                    }
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint64_t v_desc = smem_desc(sbase + C::V_OFF + st * C::V_BYTES, C::V_BYTES / 2, 1024, SWZ_128B);
                    const uint64_t pg_desc = p_desc + (uint64_t)(((k & 1) * C::P_BYTES + h * (C::P_BYTES / 2) + g * rph * 128) / 16);
                    if (leader) {
#pragma unroll
                        for (int c = 0; c < HALF / 16; ++c)
                            mma_bf16(tb + TM_O + g * rph, v_desc + (uint64_t)(c * 16 * 128 / 16), pg_desc + (uint64_t)(c * 32 / 16), idesc_o,
                                     !(p == p_lo && h == 0 && c == 0));
                        tc_commit(&X->v_empty[st]);
                    }
                    __syncwarp();
                }
                if (ok && leader) tc_commit(&X->pv_done[k & 1]);
                __syncwarp();
            }
            ++seg;
        }
        drain(leader, 1);
    } else if (VQ && warp >= 12) {
        // ================================================================== quantised values -> bf16 operand tiles
        // Every E2M1 level is a bf16 number; the token's scale goes into the softmax weight. 128 threads, two per token, eight tokens
        // side by side, so that the eight lanes of a store have the eight chunks of a swizzled line.
        const int r = (tid - 384) / 32 * 16 + (lane >> 4) * 8 + (lane & 7), part = lane >> 3 & 1;
        auto prmt = [](uint32_t a, uint32_t b, uint32_t c) -> uint32_t {
            uint32_t d;
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
            return d;
        };
        // bf16 of 0 .5 1 1.5 2 3 4 6: high bytes 00 3F 3F 3F 40 40 40 40, low bytes 00 00 80 C0 00 40 80 C0
        constexpr uint32_t HI_A = 0x3F3F3F00u, HI_B = 0x40404040u, LO_A = 0xC0800000u, LO_B = 0xC0804000u;
        int k = 0;
        bool ok = true;
        while (ok && walk.next(A.B, tl, zi, s)) {
            const int tiles = 2 * heads(s) * (s.p_hi - s.p_lo);
            for (int j = 0; j < tiles && ok; ++j, ++k) {
                const int rs = k % (C::NR ? C::NR : 1), st = k % C::NV;
                ok = wait_or_abort(&X->r_full[rs], (k / (C::NR ? C::NR : 1)) & 1, X, A.status, 50);
                if (ok && k >= C::NV) ok = wait_or_abort(&X->v_empty[st], (k / C::NV - 1) & 1, X, A.status, 51);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint8_t* raw = smem + C::R_OFF + rs * C::RAW_BYTES + r * 64;
                uint8_t* row = smem + C::V_OFF + st * C::V_BYTES + part * (C::V_BYTES / 2) + r * 128;      // 64 dims of the token
#pragma unroll
                for (int c = 0; c < 2; ++c) {                           // 32 codes -> 64 bytes
                    const uint4 w4 = *reinterpret_cast<const uint4*>(raw + (((part * 2 + c) ^ ((r >> 1) & 3)) << 4));
                    const uint32_t wv[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t w = wv[u], mag = w & 0x77777777u, up = w << 4;
                        const uint32_t h0 = prmt(HI_A, HI_B, mag) | (prmt(up, w, 0x5140u) & 0x80808080u);
                        const uint32_t h1 = prmt(HI_A, HI_B, mag >> 16) | (prmt(up, w, 0x7362u) & 0x80808080u);
                        const uint32_t l0 = prmt(LO_A, LO_B, mag), l1 = prmt(LO_A, LO_B, mag >> 16);
                        const uint4 o = make_uint4(prmt(l0, h0, 0x5140u), prmt(l0, h0, 0x7362u), prmt(l1, h1, 0x5140u), prmt(l1, h1, 0x7362u));
                        *reinterpret_cast<uint4*>(row + (((c * 4 + u) ^ (r & 7)) << 4)) = o;
                    }
                }
                fence_proxy_async_smem();
                arrive_warp(&X->v_full[st]);
                arrive_warp(&X->r_empty[rs]);
            }
        }
    } else if (warp >= 4) {
        // ================================================================== softmax: two threads per row, half of a page's tokens each
        // Both halves of a page are worked on at the same time, and the tensor core does the next page's scores meanwhile. (A page
        // per group, the groups taking turns and handing on the rows' references: 57 against 51 us for 4 x 4096 tokens of 32 kv heads,
        // 184 against 172 us for 16 x 16384 tokens of quantised values. Four groups of 32 columns: 128 against 129 us for 64 drafts, 303
        // against 298 for 16 x 32768 tokens, 16 drafts.)
        const int quad = warp & 3, grp = (warp - 4) >> 2, r = quad * 32 + lane;
        const uint32_t tl_s = tb + ((uint32_t)(quad * 32) << 16);
        const float* row_scale = reinterpret_cast<const float*>(smem + C::Q_OFF + PKV_QUERY_TERMS * C::PAGE);
        uint8_t* p_row = smem + C::P_OFF + grp * (C::P_BYTES / 2) + r * 128;
        int k = 0, kv = 0, seg = 0;
        bool ok = true;                              // false once any wait of this warp gave up; the loop ends for all warps together
        auto wait_all = [&](uint64_t* bar, uint32_t parity, int where) {
            ok = __all_sync(0xffffffffu, ok && wait_or_abort(bar, parity, X, A.status, where));
        };
        bool go = true;
        while (go && walk.next(A.B, tl, zi, s)) {
            const int ng = heads(s), base = s.T - s.n, first = s.z / s.t.groups * s.t.qpb, nq = min(s.t.qpb, s.n - first), rph = s.t.rph;
            const int gl = r / rph, rr = r % rph;
            const bool mine = gl < ng && rr < nq * tl.rep;              // a drafted token's row
            const bool busy = __any_sync(0xffffffffu, mine);
            unsigned long long word = 0;
            if (mine) {
                const int i = first + rr / tl.rep;
                word = A.mask ? (unsigned long long)A.mask[s.lo + i] : (i >= 63 ? ~0ull : (2ull << i) - 1);
                if (s.n < 64) word &= (1ull << s.n) - 1;
            }
            wait_all(&X->q_full[PKV_QUERY_TERMS - 1], seg & 1, 40);      // (the rows' scales come with the last term)
            float cs = ok ? row_scale[r] * A.col_scale : 0.0f;
            if (cs < 1e-37f) cs = 1e-37f;                               // (keeps NaN; a masked score -inf x cs stays -inf)
            arrive_warp(&X->q_empty);
            float m = -INFINITY, l = 0.0f;                              // the row's reference (both threads the same), this thread's sum
            for (int p = s.p_lo; p < s.p_hi; ++p, ++k, kv += 2 * ng) {
                const int drafts = base - p * PKV_PAGE_TOKENS, buf = k & 1;
                const bool masked = drafts < (grp + 1) * HALF;
                const uint32_t s_tm = tl_s + TM_S + 128 * buf + HALF * grp;
                float2 sum;
                const bool opening = p == s.p_lo;
                bool moved = false;
                // scores, value scales, and the weights of two pages ago read: usually all there, one vote then
                bool there = mbar_try_wait(&X->s_full[buf], (k >> 1) & 1);
                if constexpr (VQ) there = there && mbar_try_wait(&X->sc_full[buf], (k >> 1) & 1);
                if (k >= 2) there = there && mbar_try_wait(&X->pv_done[buf], ((k >> 1) - 1) & 1);
                if (!__all_sync(0xffffffffu, there)) {
                    wait_all(&X->s_full[buf], (k >> 1) & 1, 41);
                    if constexpr (VQ) wait_all(&X->sc_full[buf], (k >> 1) & 1, 46);
                    if (k >= 2) wait_all(&X->pv_done[buf], ((k >> 1) - 1) & 1, 43);
                }
                tc_fence_after_sync();
                // Weights at the reference that the row had so far, the page's maximum on the way. The reference only moves when a
                // page exceeds it by 2^8 (its column of O^T is then rescaled), so the weights are rarely formed a second time.
                // The loop is not unrolled beyond 32 columns: the code of all roles has to fit the instruction cache together, or
                // each of them runs at the speed of instruction fetch (unrolled over the 128 columns: 192 against 165 us).
#pragma unroll 1
                for (bool first_try = true;; first_try = false) {
                    const float mu = m > -INFINITY ? m : 0.0f;          // nothing seen yet: every weight is 2^-inf
                    const float2 cs2 = make_float2(cs, cs), mu2 = make_float2(-mu, -mu);
                    float top = -INFINITY;
                    sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
                    for (int c = 0; c < 2 && busy; ++c) {
                        float x[32];
                        uint32_t w[16];
                        if (ok) tmem_ld32(s_tm + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
                        tmem_ld_wait();
                        uint32_t see = 0u;
                        if (__builtin_expect(masked, false)) {                                   // tokens that the row does not see
                            const int j0 = HALF * grp + 32 * c - drafts;             // drafted token of the first column (negative: cached)
                            see = j0 >= 0 ? (j0 < 64 ? (uint32_t)(word >> j0) : 0u) : (j0 > -32 ? (uint32_t)(word << -j0) | ((1u << -j0) - 1) : ~0u);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(see >> e & 1)) x[e] = -INFINITY;
                        }
                        float mx[2] = {top, x[0]};
#pragma unroll
                        for (int e = 1; e < 31; e += 2) mx[(e >> 1) & 1] = max3(mx[(e >> 1) & 1], x[e], x[e + 1]);
                        top = max3(mx[0], mx[1], x[31]);
                        if (opening && first_try) continue;             // no reference yet: the maximum alone
                        if constexpr (VQ) {
                            // The weight of a token carries its value scale of this row's kv head, and the product is rounded to bf16
                            // (2^-8 of it); the sum takes the weights themselves, which the scale is no part of.
                            const uint4* sc = reinterpret_cast<const uint4*>(smem + C::SC_OFF + buf * C::SC_BYTES + min(gl, ng - 1) * PKV_PAGE_TOKENS * 2 + (2 * grp + c) * 64);
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const uint4 q4 = sc[u];
                                const uint32_t qs[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float2 t = fma2(make_float2(x[8 * u + 2 * e], x[8 * u + 2 * e + 1]), cs2, mu2);
                                    t = make_float2(ex2_fast(t.x), ex2_fast(t.y));
                                    sum = add2(sum, t);
                                    t = mul2(t, make_float2(__uint_as_float(qs[e] << 16), __uint_as_float(qs[e] & 0xffff0000u)));
                                    w[4 * u + e] = pack_bf16(t.x, t.y);
                                }
                            }
                            if (masked) {                               // a masked token's scale may be anything
#pragma unroll
                                for (int e = 0; e < 16; ++e) w[e] &= (see >> (2 * e) & 1 ? 0xffffu : 0u) | (see >> (2 * e) & 2 ? 0xffff0000u : 0u);
                            }
                        } else {
                            // rounded to bf16 for the tensor core (2^-8 of a weight at most, up as often as down); the sum takes the weights
                            // themselves (over what was rounded it takes 3 % longer: 138 against 134 us for 64 drafts). Five of 16 pairs
                            // go to the multiply-add units (2, 4 or 8: slower): 8 x 8192 tokens, 64 drafts take 125 us instead of 129 in
                            // short runs, 135.6 instead of 137.1 in long ones at the power limit; 128 columns 110.6 instead of 114.2 and 114.4
                            // instead of 115.3. Tiles of several kv heads wait for values and for power: none (16 x 16384 tokens, 16 drafts,
                            // 128 columns: 119 and 134 us with none, 122 and 140 with five; 4 x 16384, 32 kv heads: 106.0 and 106.4).
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                float2 t = fma2(make_float2(x[2 * e], x[2 * e + 1]), cs2, mu2);
                                t = !MANY && e % 3 == 2 ? ex2_cubic(t) : make_float2(ex2_fast(t.x), ex2_fast(t.y));
                                w[e] = pack_bf16(t.x, t.y);
                                sum = add2(sum, t);
                            }
                        }
                        // P: row r, 64 tokens of 16 bit per 128-byte swizzled line, a block per half page
                        uint8_t* line = p_row + buf * C::P_BYTES;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            *reinterpret_cast<uint4*>(line + (((c * 4 + u) ^ (r & 7)) << 4)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
                    }
                    fence_proxy_async_smem();
                    if (!first_try) break;
                    top = mine ? top * cs : -INFINITY;                  // (a row that nobody has: whatever its column becomes, nobody reads it)
                    if (__builtin_expect(!opening && !softmax_any(top > m + RESCALE_THRESHOLD || !ok), true)) break;
                    if (softmax_any(!ok)) { go = false; break; }
                    moved = true;
                    X->row_l[grp][r] = top;
                    softmax_sync();
                    top = fmaxf(top, X->row_l[grp ^ 1][r]);
                    const float now = top > m + RESCALE_THRESHOLD ? top : m, f = now != m ? exp2f(m - now) : 1.0f;
                    if (grp == 0) X->row_f[0][r] = f;
                    l *= f;
                    const bool again = opening || __any_sync(0xffffffffu, now != m);
                    m = now;
                    if (!again) break;
                }
                if (!go) break;
                tc_fence_before_sync();
                arrive_warp(&X->s_empty[buf]);
                if constexpr (VQ) arrive_warp(&X->sc_empty[buf]);
                l += sum.x + sum.y;
                if (__builtin_expect(moved, false)) {
                    softmax_sync();                                     // row_f is there; row_l may be written again
                    if (!opening) {
                        wait_all(&X->pv_done[buf ^ 1], ((k - 1) >> 1) & 1, 49);         // the accumulators are at rest
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int c0 = 16 * grp; c0 < ng * rph; c0 += 32) {
                            uint32_t o[16];
                            tmem_ld16(tl_s + TM_O + c0, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * X->row_f[0][c0 + c]);
                            tmem_st16(tl_s + TM_O + c0, o);
                        }
                        tmem_st_wait();
                        tc_fence_before_sync();
                    }
                }
                arrive_warp(&X->p_full[buf]);
                if constexpr (!VQ) {
                    // Values behind the cached tokens: rows past the sequence become zero, and so does what is not finite in a
                    // drafted row (0 x inf would reach rows that do not see it); who does see it gets NaN at the end.
                    if (__builtin_expect(drafts < PKV_PAGE_TOKENS && ok, false)) {
                        if (k > 0) wait_all(&X->pv_done[buf ^ 1], ((k - 1) >> 1) & 1, 50);
                        // (Every tile of such a page is handed over, also one with cached rows only: the page before is known to be
                        // consumed, and within this one the stages then advance in step with these waits.)
                        for (int j = 0; j < 2 * ng; ++j) {
                            const int h = j & 1, st = (kv + j) % C::NV;
                            wait_all(&X->v_full[st], ((kv + j) / C::NV) & 1, 47);
                            if (!ok) break;
                            uint8_t* tile = smem + C::V_OFF + st * C::V_BYTES;
#pragma unroll 4
                            for (int it = 0; it < C::V_BYTES / 32 / GROUP && drafts < (h + 1) * HALF; ++it) {
                                const int id = (2 * it + grp) * GROUP + r, d = h * HALF + ((id >> 3) & 63) - drafts;      // drafted token of the row
                                if (d < 0) continue;
                                uint4* at = reinterpret_cast<uint4*>(tile) + id;
                                if (d >= s.n) { *at = make_uint4(0u, 0u, 0u, 0u); continue; }
                                uint4 v = *at;
                                uint32_t* e = reinterpret_cast<uint32_t*>(&v);
                                bool hit = false;
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    if ((e[q] & 0x7f80u) == 0x7f80u) { e[q] &= 0xffff0000u; hit = true; }
                                    if ((e[q] & 0x7f800000u) == 0x7f800000u) { e[q] &= 0xffffu; hit = true; }
                                }
                                if (hit) { *at = v; atomicOr(&X->bad[seg % 3][j >> 1][d >> 5], 1u << (d & 31)); }
                            }
                            fence_proxy_async_smem();
                            arrive_warp(&X->v_clean[st]);
                        }
                    }
                }
            }
            if (!go) break;
            // ---- the tile's stretch is done: O^T out of tensor memory, 64 columns by each group
            wait_all(&X->pv_done[(k - 1) & 1], ((k - 1) >> 1) & 1, 44);
            X->row_l[grp][r] = l;
            if (r < MAX_G * 2) (&X->bad[(seg + 1) % 3][0][0])[r] = 0u;  // (last read two stretches ago)
            if (softmax_any(!ok)) { go = false; break; }
            tc_fence_after_sync();
            const bool whole = s.p_lo == 0 && s.p_hi == s.pages;
            const size_t slot = (size_t)blockIdx.x * 2 + (s.p_lo == 0);
            l = X->row_l[0][r] + X->row_l[1][r];
            if (!VQ && mine && ((word & 0xffffffffu & X->bad[seg % 3][gl][0]) | ((word >> 32) & X->bad[seg % 3][gl][1]))) l = __int_as_float(0x7fc00000);
            X->row_f[grp][r] = l == 0.0f ? 0.0f : 1.0f / l;             // a row that sees nothing: zeros
            X->row_o[grp][r] = mine ? (s.lo + first + rr / tl.rep) * A.n_q + (s.z % s.t.groups * s.t.G + gl) * tl.rep + rr % tl.rep : -1;
            if (!whole && mine && grp == 0) A.part_ml[slot * ROWS + r] = make_float2(m, l);
            group_sync(grp);
            // (16 columns at a time in a rolled loop: this thread's dim is r)
#pragma unroll 1
            for (int c0 = 64 * grp; c0 < min(ng * rph, 64 * grp + 64); c0 += 16) {
                uint32_t o[16];
                tmem_ld16(tl_s + TM_O + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int c4 = 0; c4 < 16; c4 += 4) {
                    const int4 t4 = *reinterpret_cast<const int4*>(&X->row_o[grp][c0 + c4]);
                    const float4 f4 = *reinterpret_cast<const float4*>(&X->row_f[grp][c0 + c4]);
                    const int to[4] = {t4.x, t4.y, t4.z, t4.w};
                    const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (to[c] < 0) continue;
                        if (whole) A.out[(size_t)to[c] * DH + r] = __float2bfloat16(__uint_as_float(o[c4 + c]) * f[c]);
                        else A.part_o[(slot * ROWS + c0 + c4 + c) * DH + r] = __uint_as_float(o[c4 + c]);
                    }
                }
            }
            tc_fence_before_sync();
            arrive_warp(&X->o_empty);
            group_sync(grp);                                            // row_f, row_o are free again
            ++seg;
        }
    }
    // ---- everyone meets, tensor memory goes back
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 3) tmem_dealloc(tb, TM_COLS);
    if (X->abort_flag) {                             // a stretch that was not finished counts for nothing in the merge
        for (int i = tid; i < 2 * ROWS; i += C::NTHREADS) A.part_ml[(size_t)blockIdx.x * 2 * ROWS + i] = make_float2(-INFINITY, 0.0f);
    }
}

// ------------------------------------------------------------------------------------------------ merge
// O = sum 2^(m - M) o / sum 2^(m - M) l over the stretches of a tile that several gangs had. A warp has RW rows (a lane four dims of
// each); WPR warps share the stretches of their rows. References, sums and outputs of DEEP stretches are asked for together: many
// rows of few stretches, or few rows of many. Latency and the launch itself (one sequence in 74 stretches: 5 us).
template <int WPR, int RW, int DEEP>
__global__ void __launch_bounds__(256) pkv_tree_merge_kernel(const AttnArgs A) {
    __shared__ float4 acc_s[WPR > 1 ? 8 : 1][RW][32];
    __shared__ float2 ml_s[8][RW];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, z = blockIdx.y, b = blockIdx.z;
    const int r0 = (blockIdx.x * (8 / WPR) + warp / WPR) * RW, w0 = warp % WPR;
    const Tiles& X = A.X;
    pkv_grid_launch_dependents();
    pkv_grid_wait();
    int lo, n, T;
    const int pages = A.B.pages(b, lo, n, T), U = A.first_page[A.B.batch], gang = A.first_page[A.B.batch + 1], gangs = A.first_page[A.B.batch + 2];
    const int list = A.first_page[b];
    if (pages == 0) return;
    const Shape t = X.of(n);
    if (z >= t.Z) return;
    const int cost = cost_of(t, gang), u0 = list + (gang ? z / gang : z) * pages * cost, zi = gang ? z % gang : 0;
    const Cut cut(U, gangs);
    const int x0 = cut.of(u0), x1 = cut.of(u0 + (pages - 1) * cost);
    if (x0 == x1) return;                            // one CTA did the whole tile and has written it
    const int gl = r0 / t.rph, rr0 = r0 % t.rph, g = z % t.groups * t.G + gl, first = z / t.groups * t.qpb;      // (rph is a multiple of 16)
    const int rows = gl < t.G && g < A.n_kv ? min(RW, min(t.qpb, n - first) * X.rep - rr0) : 0;
    float M[RW], l[RW];
    float4 acc[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) { M[r] = -INFINITY; l[r] = 0.0f; acc[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    if (rows > 0) {
#pragma unroll 1
        for (int xb = x0 + w0; xb <= x1; xb += WPR * DEEP) {
            float4 o[DEEP][RW];
            float2 ml[DEEP][RW];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int x = xb + k * WPR;
                const size_t slot = ((size_t)(gang ? x * gang + zi : x) * 2 + (x == x0)) * ROWS + r0;
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    const bool there = x <= x1 && r < rows;
                    ml[k][r] = there ? A.part_ml[slot + r] : make_float2(-INFINITY, 0.0f);
                    if (there) o[k][r] = reinterpret_cast<const float4*>(A.part_o + (slot + r) * DH)[lane];
                }
            }
#pragma unroll
            for (int k = 0; k < DEEP; ++k)
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    if (ml[k][r].x == -INFINITY) {       // (a stretch that saw nothing of the row: zeros, or NaN in the sum)
                        l[r] += ml[k][r].y;
                        continue;
                    }
                    const float top = fmaxf(M[r], ml[k][r].x), was = exp2f(M[r] - top), now = exp2f(ml[k][r].x - top);
                    M[r] = top;
                    l[r] = fmaf(l[r], was, ml[k][r].y * now);
                    acc[r].x = fmaf(acc[r].x, was, o[k][r].x * now); acc[r].y = fmaf(acc[r].y, was, o[k][r].y * now);
                    acc[r].z = fmaf(acc[r].z, was, o[k][r].z * now); acc[r].w = fmaf(acc[r].w, was, o[k][r].w * now);
                }
        }
    }
    if constexpr (WPR > 1) {                         // the first of the WPR warps adds the others' sums to its own
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            acc_s[warp][r][lane] = acc[r];
            if (lane == 0) ml_s[warp][r] = make_float2(M[r], l[r]);
        }
        __syncthreads();
        if (w0 != 0) return;
#pragma unroll 1
        for (int w = 1; w < WPR; ++w)
#pragma unroll
            for (int r = 0; r < RW; ++r) {
                const float2 ml = ml_s[warp + w][r];
                const float4 o = acc_s[warp + w][r][lane];
                if (ml.x == -INFINITY) { l[r] += ml.y; continue; }
                const float top = fmaxf(M[r], ml.x), was = exp2f(M[r] - top), now = exp2f(ml.x - top);
                M[r] = top;
                l[r] = fmaf(l[r], was, ml.y * now);
                acc[r].x = fmaf(acc[r].x, was, o.x * now); acc[r].y = fmaf(acc[r].y, was, o.y * now);
                acc[r].z = fmaf(acc[r].z, was, o.z * now); acc[r].w = fmaf(acc[r].w, was, o.w * now);
            }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r) {
        if (r >= rows) continue;
        const float f = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        const size_t row = (size_t)(lo + first + (rr0 + r) / X.rep) * A.n_q + g * X.rep + (rr0 + r) % X.rep;
        *reinterpret_cast<uint2*>(A.out + row * DH + lane * 4) = make_uint2(pack_bf16(acc[r].x * f, acc[r].y * f), pack_bf16(acc[r].z * f, acc[r].w * f));
    }
}

// ------------------------------------------------------------------------------------------------ host
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

int init_encoder() {
    if (!g_encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        PKV_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
        if (!fn || qres != cudaDriverEntryPointSuccess) return PKV_ERR_CUDA;
        g_encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
    return PKV_OK;
}

// rows of 128 bytes, or (bf16) of 128 values in two boxes of 64 with the 128-byte swizzle
int encode_map(CUtensorMap* map, const void* base, uint64_t rows, uint32_t box_rows, bool bf16) {
    cuuint64_t dims[2] = {128, rows};
    cuuint64_t strides[1] = {(cuuint64_t)(bf16 ? 256 : 128)};
    cuuint32_t box[2] = {(cuuint32_t)(bf16 ? 64 : 128), box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = g_encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
                          estr, CU_TENSOR_MAP_INTERLEAVE_NONE, bf16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { g_pkv_last_cuda_error = (int)r; return PKV_ERR_CUDA; }
    return PKV_OK;
}

// Rows of a kv head: rep query heads of up to qpb drafted tokens, in blocks of equal size when there are more than 128; padded
// to the 16 columns an MMA takes. As many kv heads per tile as fit, evenly over the tiles.
Tiles make_tiles(int n_q, int n_kv, int max_draft, bool quantised) {
    Tiles X;
    X.quantised = quantised;
    X.rep = n_q / n_kv;
    X.rep_inv = 65536 / X.rep + 1;                   // (rows below 128, rep <= 64: 128 / 65536 < 1 / 64)
    X.Z = 1;
    X.shape[0] = 0;
    const int most = ROWS / X.rep;
    for (int n = 1; n <= PKV_TREE_MAX; ++n) {
        const int blocks = (n + most - 1) / most, qpb = (n + blocks - 1) / blocks, rph = (X.rep * qpb + 15) / 16 * 16;
        const int fit = ROWS / rph, even = (n_kv + fit - 1) / fit, G = (n_kv + even - 1) / even, groups = (n_kv + G - 1) / G;
        X.shape[n] = (uint32_t)(qpb - 1) | (uint32_t)(rph / 16 - 1) << 6 | (uint32_t)(G - 1) << 9 | (uint32_t)(groups - 1) << 12;
        if (n <= max_draft && groups * blocks > X.Z) X.Z = groups * blocks;
    }
    return X;
}

struct Layout { size_t blobs, part_o, part_ml, first_page, total; };

Layout make_layout(const Tiles& X, int batch, int WP) {
    Layout y;
    const size_t ctas = N_SM;
    y.blobs = 0;
    y.part_o = ((size_t)batch * X.Z * blob_bytes(WP) + 1023) / 1024 * 1024;
    y.part_ml = y.part_o + ctas * 2 * ROWS * DH * 4;
    y.first_page = y.part_ml + ctas * 2 * ROWS * 8;
    y.total = y.first_page + ((size_t)batch + 3) * 4;
    return y;
}

template <int WP, bool VQ, bool MANY>
int launch(const pkv_cache_t* cache, const AbsorbArgs& ab, const AttnArgs& at, size_t blob_rows, cudaStream_t st) {
    using C = Cfg<WP, VQ, MANY>;
    const Tiles& X = ab.X;
    CUtensorMap kmap, qmap, vmap;
    int rc = encode_map(&kmap, cache->latent_dev, (uint64_t)cache->n_pages * (C::PAGE / 128), C::PAGE / 128, false);
    if (!rc) rc = encode_map(&qmap, ab.blobs, blob_rows, C::PAGE / 128, false);
    if (!rc) rc = VQ ? encode_map(&vmap, cache->vq_dev, (uint64_t)cache->n_pages * cache->n_kv * (PKV_VQ_TILE_BYTES / 128), C::RAW_BYTES / 128, false)
                     : encode_map(&vmap, cache->v_dev, (uint64_t)cache->n_pages * cache->n_kv * PKV_PAGE_TOKENS, HALF, true);
    if (rc) return rc;
    static pkv_attr_flags attr;
    PKV_CUDA_TRY(pkv_set_max_smem(pkv_tree_attn_kernel<WP, VQ, MANY>, C::SMEM, attr));
    PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_absorb_kernel<WP>, dim3(ROWS / AR + 1, X.Z, ab.B.batch), dim3(AR * WP / 16), 0, st, ab));
    PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_attn_kernel<WP, VQ, MANY>, dim3(N_SM), dim3(C::NTHREADS), C::SMEM, st, kmap, qmap, vmap, at));
    // Stretches of a tile, if all sequences have as many tiles and pages: the more, the more warps share a row's. The three forms, all
    // launches together: 3 stretches (16 x 32768 tokens, 16 drafts) 299, 304 and 345 us; 6 (7 x 20000, 16) 92, 95 and 121; 10 (4 x 4096,
    // 32 kv heads, 8) 54, 49 and 61; 75 (131072, 8) 108, 79 and 69.
    const int parts = N_SM / (ab.B.batch * X.Z) + 1;
    const dim3 block(256);
    if (parts <= 6) PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_merge_kernel<1, 4, 2>, dim3(ROWS / 32, X.Z, ab.B.batch), block, 0, st, at));
    else if (parts <= 16) PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_merge_kernel<2, 1, 8>, dim3(ROWS / 4, X.Z, ab.B.batch), block, 0, st, at));
    else PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_merge_kernel<8, 1, 10>, dim3(ROWS, X.Z, ab.B.batch), block, 0, st, at));
    return PKV_OK;
}

int check_shape(const pkv_layer_t* L, int32_t batch, int32_t max_draft, int32_t max_pages) {
    int st = pkv_check_layer(L);
    if (st) return st;
    if (batch < 0 || max_draft <= 0 || max_pages <= 0) return PKV_ERR_INVALID;
    if (L->head_dim != DH || max_draft > PKV_TREE_MAX || L->n_q / L->n_kv > 64 || batch > 4096 || max_pages > (1 << 23)) return PKV_ERR_UNSUPPORTED;
    return PKV_OK;
}

}  // namespace

extern "C" int64_t pkv_tree_workspace_bytes(const pkv_layer_t* layer, int32_t batch, int32_t max_draft, int32_t max_pages) {
    int st = check_shape(layer, batch, max_draft, max_pages);
    if (st) return st;
    return (int64_t)make_layout(make_tiles(layer->n_q, layer->n_kv, max_draft, false), batch, pkv_padded_width(2 * layer->R + layer->R_s)).total;
}

extern "C" int pkv_tree_attn(const pkv_layer_t* layer, const pkv_cache_t* cache, const pkv_pages_t* pages, const void* q_dev, int32_t q_dtype,
                             const int32_t* positions_dev, const int64_t* mask_dev, const int32_t* cu_dev, int32_t n_tokens,
                             int32_t max_draft, void* workspace_dev, int64_t workspace_bytes, void* out_dev, int32_t* status_dev,
                             void* stream) {
    if (!pages || !pages->page_table_dev || !pages->seqlens_dev || n_tokens < 0) return PKV_ERR_INVALID;
    int st = check_shape(layer, pages->batch, max_draft, pages->max_pages);
    if (st) return st;
    st = pkv_check_cache(cache);
    if (st) return st;
    if (cache->W != 2 * layer->R + layer->R_s || cache->n_kv != layer->n_kv || cache->head_dim != layer->head_dim) return PKV_ERR_INVALID;
    const void* v = cache->v_bits ? cache->vq_dev : cache->v_dev;
    if (!v || (((uintptr_t)v) & (cache->v_bits ? 127u : 15u))) return PKV_ERR_INVALID;
    if (q_dtype != PKV_F32 && q_dtype != PKV_BF16) return PKV_ERR_UNSUPPORTED;
    if (pages->batch == 0 || n_tokens == 0) return PKV_OK;
    if (!q_dev || !positions_dev || !cu_dev || !out_dev || (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15u)) return PKV_ERR_INVALID;
    const int WP = pkv_padded_width(cache->W);
    // coordinates of the tensor maps are 31 bits
    if ((int64_t)cache->n_pages * cache->n_kv * PKV_PAGE_TOKENS > 0x7fffffff || (int64_t)cache->n_pages * 144 > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
    const Tiles X = make_tiles(layer->n_q, layer->n_kv, max_draft, cache->v_bits != 0);
    const Layout y = make_layout(X, pages->batch, WP);
    const size_t blob_rows = (size_t)pages->batch * X.Z * (blob_bytes(WP) / 128);
    if (blob_rows > 0x7fffffff || X.Z > 65535 || (int64_t)pages->batch * pages->max_pages * X.Z > 0x3fffffff / COST_MOST) return PKV_ERR_UNSUPPORTED;
    if ((int64_t)n_tokens * layer->n_q > 0x7fffffff) return PKV_ERR_UNSUPPORTED;      // rows of the result are 31 bits
    if (!workspace_dev || (((uintptr_t)workspace_dev) & 1023u) || workspace_bytes < (int64_t)y.total) return PKV_ERR_INVALID;
    st = init_encoder();
    if (st) return st;
    uint8_t* ws = (uint8_t*)workspace_dev;
    const Batch B{cu_dev, pages->seqlens_dev, pages->batch, pages->max_pages, n_tokens, max_draft};
    const AbsorbArgs ab{*layer, B, X, q_dev, q_dtype == PKV_BF16, positions_dev, ws, (int32_t*)(ws + y.first_page), status_dev};
    AttnArgs at;
    at.B = B; at.X = X; at.page_table = pages->page_table_dev; at.mask = mask_dev; at.blobs = ws; at.vq = (const uint8_t*)cache->vq_dev;
    at.n_pages = cache->n_pages; at.n_kv = layer->n_kv; at.n_q = layer->n_q;
    at.col_scale = layer->second * PKV_LOG2E / sqrtf((float)DH);
    at.part_o = (float*)(ws + y.part_o); at.part_ml = (float2*)(ws + y.part_ml); at.first_page = (int32_t*)(ws + y.first_page);
    at.out = (__nv_bfloat16*)out_dev; at.status = status_dev;
    cudaStream_t s = (cudaStream_t)stream;
    if (cache->v_bits) return WP == 256 ? launch<256, true, false>(cache, ab, at, blob_rows, s) : launch<128, true, false>(cache, ab, at, blob_rows, s);
    // kv heads of the largest tree's tiles: the call's own lengths are on the device (16 x 16384 tokens, 6 drafts: 121 us in a workspace for
    // 6 or 16, 135 in one for 64)
    const bool many = (X.shape[max_draft] >> 9 & 7u) > 0;
    if (WP == 128) return many ? launch<128, false, true>(cache, ab, at, blob_rows, s) : launch<128, false, false>(cache, ab, at, blob_rows, s);
    return many ? launch<256, false, true>(cache, ab, at, blob_rows, s) : launch<256, false, false>(cache, ab, at, blob_rows, s);
}
