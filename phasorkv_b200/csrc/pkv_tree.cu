// Attention of a tree of drafted tokens over the paged latent cache.
//
//   S[i, h, t] = q'_{i,h} . c_t,   O[i, h] = softmax_t(S d^-1/2) V_{g(h)}   over t < base and t = base + j, bit j of mask_i
//
// with q' the absorbed query of drafted token i (conj(A) zq e^{i theta pos}; slow dims unrotated) and c_t the NVFP4 rows.
// First form, on the CUDA cores: a CTA takes one drafted token, one kv head and up to eight of its query heads and
// walks the sequence page by page, a token per thread for the scores, a dim per thread for P.V.
#include "pkv_common.cuh"

int pkv_check_layer(const pkv_layer_t* L);
int pkv_check_cache(const pkv_cache_t* c);

namespace {

constexpr int DH = 128, NT = 128, RC = 8;

struct Args {
    pkv_layer_t L;
    pkv_cache_t C;
    pkv_pages_t pg;
    const void* q;
    int q_bf16, n_tokens, max_draft;
    const int32_t *positions, *cu;
    const int64_t* mask;
    __nv_bfloat16* out;
    int32_t* status;
};

__global__ void __launch_bounds__(NT) pkv_tree_attn_kernel(const Args A) {
    __shared__ float qa[RC][PKV_MAX_WIDTH];
    __shared__ float qs[RC][DH];
    __shared__ float2 ph[DH / 2];
    __shared__ float ps[RC][NT];
    __shared__ float red[RC][4];
    const pkv_layer_t& L = A.L;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.y;
    const int rep = L.n_q / L.n_kv, r0 = blockIdx.z * RC, nr = min(RC, rep - r0), W = A.C.W;
    pkv_grid_launch_dependents();
    pkv_grid_wait();
    const int i = blockIdx.x;
    int b = 0;
    while (b < A.pg.batch && A.cu[b + 1] <= i) ++b;
    if (b == A.pg.batch) return;
    const int lo = A.cu[b], n = A.cu[b + 1] - lo, T = A.pg.seqlens_dev[b], base = T - n, row = i - lo;
    if (lo < 0 || row < 0 || A.cu[b + 1] > A.n_tokens || n > A.max_draft || base < 0 || T > A.pg.max_pages * PKV_PAGE_TOKENS) {
        if (A.status && tid == 0) { atomicExch(&A.status[0], 4); atomicExch(&A.status[1], b); }
        return;
    }
    const unsigned long long word = A.mask ? (unsigned long long)A.mask[i] : (row >= 63 ? ~0ull : (2ull << row) - 1);
    for (int k = tid; k < nr * DH; k += NT) {
        const size_t o = ((size_t)i * L.n_q + g * rep + r0 + k / DH) * DH + k % DH;
        qs[k / DH][k % DH] = A.q_bf16 ? __bfloat162float(((const __nv_bfloat16*)A.q)[o]) : ((const float*)A.q)[o];
    }
    for (int j = tid; j < DH / 2; j += NT) {
        double sn, cs;
        sincos((double)A.positions[i] * L.inv_freq_dev[j], &sn, &cs);
        ph[j] = make_float2((float)(L.attn_scale * cs), (float)(L.attn_scale * sn));
    }
    __syncthreads();
    for (int k = tid; k < nr * W; k += NT) {
        const int r = k / W, c = k % W;
        float v = 0.0f;
        if (c < 2 * L.R) {
            const int d = c < L.R ? c : c - L.R, f = L.freq_dev[d];
            const float zr = qs[r][f] * ph[f].x - qs[r][f + DH / 2] * ph[f].y, zi = qs[r][f] * ph[f].y + qs[r][f + DH / 2] * ph[f].x;
            const float ar = L.A_re_dev[g * L.R + d], ai = L.A_im_dev[g * L.R + d];
            v = c < L.R ? ar * zr + ai * zi : ar * zi - ai * zr;
        } else {
            for (int s = 0; s < 2 * L.n_slow; ++s)
                v = fmaf(qs[r][s < L.n_slow ? L.slow_dev[s] : L.slow_dev[s - L.n_slow] + DH / 2],
                         L.A_s_dev[((size_t)g * 2 * L.n_slow + s) * L.R_s + c - 2 * L.R], v);
        }
        qa[r][c] = v * (PKV_LOG2E * rsqrtf((float)DH)) * (L.second_blocks_dev ? L.second_blocks_dev[c >> 4] : L.second);
    }
    float m[RC], l[RC], acc[RC];
    for (int r = 0; r < RC; ++r) { m[r] = -INFINITY; l[r] = acc[r] = 0.0f; }
    const int RB = pkv_row_bytes(W), pb = pkv_page_bytes(W);
    for (int p = 0; p * PKV_PAGE_TOKENS < T; ++p) {
        const int page = A.pg.page_table_dev[(size_t)b * A.pg.max_pages + p];
        if (page < 0 || page >= A.C.n_pages) {
            if (A.status && tid == 0) { atomicExch(&A.status[0], 2); atomicExch(&A.status[1], p); }
            return;
        }
        const int t = p * PKV_PAGE_TOKENS + tid;
        const bool see = t < base || (t < T && (word >> (t - base) & 1));
        float s[RC] = {};
        const uint8_t* pg = A.C.latent_dev + (size_t)page * pb;
        __syncthreads();
        for (int j = 0; j < W / 16; ++j) {
            const uint2 w = *reinterpret_cast<const uint2*>(pg + pkv_code_offset(tid, j * 8, RB));
            const float sc = pkv_e4m3_to_float(pg[PKV_PAGE_TOKENS * RB + pkv_scale_offset(tid, j)]);
            for (int e = 0; e < 16; ++e) {
                const float c = pkv_e2m1_value(((e < 8 ? w.x : w.y) >> (4 * (e & 7))) & 15u) * sc;
#pragma unroll
                for (int r = 0; r < RC; ++r) s[r] = fmaf(qa[r < nr ? r : 0][j * 16 + e], c, s[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < RC; ++r) {
            float x = see ? s[r] : -INFINITY;
            s[r] = x;
            for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
            if (lane == 0) red[r][warp] = x;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RC; ++r) {
            const float mn = fmaxf(m[r], fmaxf(fmaxf(red[r][0], red[r][1]), fmaxf(red[r][2], red[r][3])));
            const float f = m[r] > -INFINITY ? exp2f(m[r] - mn) : 1.0f;
            m[r] = mn; l[r] *= f; acc[r] *= f;
            ps[r][tid] = see ? exp2f(s[r] - mn) : 0.0f;
        }
        __syncthreads();
        const uint8_t* vq = (const uint8_t*)A.C.vq_dev + (size_t)page * L.n_kv * PKV_VQ_TILE_BYTES;
        const __nv_bfloat16* v = (const __nv_bfloat16*)A.C.v_dev + ((size_t)page * L.n_kv + g) * PKV_PAGE_TOKENS * DH;
        for (int k = 0; k < PKV_PAGE_TOKENS && p * PKV_PAGE_TOKENS + k < T; ++k) {
            const int tt = p * PKV_PAGE_TOKENS + k;
            if (tt >= base && !(word >> (tt - base) & 1)) continue;              // a masked row's values are never read
            float x;
            if (A.C.v_bits) {
                const uint8_t byte = vq[g * 8192 + k * 64 + ((((tid >> 1) >> 4) ^ ((k >> 1) & 3)) << 4) + ((tid >> 1) & 15)];
                x = pkv_e2m1_value(tid & 1 ? byte >> 4 : byte & 15u) *
                    __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(vq + L.n_kv * 8192 + g * 256 + k * 2));
            } else {
                x = __bfloat162float(v[k * DH + tid]);
            }
#pragma unroll
            for (int r = 0; r < RC; ++r) { acc[r] = fmaf(ps[r][k], x, acc[r]); l[r] += ps[r][k]; }
        }
    }
    for (int r = 0; r < nr; ++r)
        A.out[((size_t)i * L.n_q + g * rep + r0 + r) * DH + tid] = __float2bfloat16(m[r] > -INFINITY || l[r] != 0.0f ? acc[r] / l[r] : 0.0f);
}

}  // namespace

extern "C" int64_t pkv_tree_workspace_bytes(const pkv_layer_t* layer, int32_t batch, int32_t max_draft, int32_t max_pages) {
    if (!layer || batch < 0 || max_draft <= 0 || max_pages <= 0) return PKV_ERR_INVALID;
    if (max_draft > PKV_TREE_MAX) return PKV_ERR_UNSUPPORTED;
    return 0;
}

extern "C" int pkv_tree_attn(const pkv_layer_t* layer, const pkv_cache_t* cache, const pkv_pages_t* pages, const void* q_dev, int32_t q_dtype,
                             const int32_t* positions_dev, const int64_t* mask_dev, const int32_t* cu_dev, int32_t n_tokens,
                             int32_t max_draft, void* workspace_dev, int64_t workspace_bytes, void* out_dev, int32_t* status_dev,
                             void* stream) {
    int st = pkv_check_layer(layer);
    if (st) return st;
    st = pkv_check_cache(cache);
    if (st) return st;
    if (!pages || !pages->page_table_dev || !pages->seqlens_dev || pages->batch < 0 || pages->max_pages <= 0 || n_tokens < 0 || max_draft <= 0)
        return PKV_ERR_INVALID;
    if (cache->W != 2 * layer->R + layer->R_s || cache->n_kv != layer->n_kv || cache->head_dim != layer->head_dim) return PKV_ERR_INVALID;
    if (layer->head_dim != DH || max_draft > PKV_TREE_MAX || layer->n_q / layer->n_kv > 64 || pages->batch > 4096) return PKV_ERR_UNSUPPORTED;
    if (!(cache->v_bits ? cache->vq_dev : cache->v_dev)) return PKV_ERR_INVALID;
    if (q_dtype != PKV_F32 && q_dtype != PKV_BF16) return PKV_ERR_UNSUPPORTED;
    if (pages->batch == 0 || n_tokens == 0) return PKV_OK;
    if (!q_dev || !positions_dev || !cu_dev || !out_dev || (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15u)) return PKV_ERR_INVALID;
    Args A{*layer, *cache, *pages, q_dev, q_dtype == PKV_BF16, n_tokens, max_draft, positions_dev, cu_dev, mask_dev, (__nv_bfloat16*)out_dev, status_dev};
    const int rep = layer->n_q / layer->n_kv;
    PKV_CUDA_TRY(pkv_launch_chained(pkv_tree_attn_kernel, dim3(n_tokens, layer->n_kv, (rep + RC - 1) / RC), dim3(NT), 0, (cudaStream_t)stream, A));
    return PKV_OK;
}
