// Attention of drafted trees over a paged cache.
#include <algorithm>

#include "attn_common.h"
#include "paged.h"

namespace {

// One (row, head) by a workgroup of 256: keys [lo, hi) that the view sees.
template <class View>
__device__ void attend_one(const View& view, const int32_t* q, int32_t* out, uint32_t lo, uint32_t hi, uint32_t hd,
                           int scaled, uint32_t scale, int32_t* scores) {
    __shared__ int32_t s_q[ATTN_MAX_HEAD_DIM];
    __shared__ ArgMax s_am[4];
    __shared__ int64_t s_sum[4];
    __shared__ int32_t s_w[4];
    __shared__ int32_t s_tile[256];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (uint32_t d = tid; d < hd; d += 256) s_q[d] = q[d];
    __syncthreads();
    ArgMax best{INT32_MIN, 0xffffffffu};
    for (uint32_t j = lo + tid; j < hi; j += 256) {
        if (!view.sees(j)) continue;
        const int32_t* k = view.key(j);
        uint64_t acc = 0;
        for (uint32_t d = 0; d < hd; d++) acc += (uint64_t)((int64_t)s_q[d] * k[d]);
        const int32_t sc = scaled ? dn::scaled_score_from_sum((int64_t)acc, scale) : dn::requantize((int64_t)acc);
        scores[j - lo] = sc;
        best = argmax_combine(best, ArgMax{sc, j});
    }
    best = wave_argmax(best);
    if (lane == 0) s_am[wave] = best;
    __syncthreads();
    for (int w = 0; w < 4; w++) best = argmax_combine(best, s_am[w]);
    int64_t part = 0;
    for (uint32_t j = lo + tid; j < hi; j += 256) {
        if (!view.sees(j)) continue;
        part += (int64_t)dn::softmax_exp_diff((uint32_t)best.v - (uint32_t)scores[j - lo]);
    }
    part = wave_sum_sat64(part);
    if (lane == 0) s_sum[wave] = part;
    __syncthreads();
    const uint64_t total = (uint64_t)(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);
    const double w_scale = 65536.0 / (double)total, q_scale = 4294967296.0 / (double)total;
    int32_t wsum = 0;
    uint64_t acc[2] = {0, 0};
    for (uint32_t base = lo; base < hi; base += 256) {
        const uint32_t j = base + tid;
        int32_t w = 0;
        if (j < hi && view.sees(j))
            w = dn::softmax_weight_fast(dn::softmax_exp_diff((uint32_t)best.v - (uint32_t)scores[j - lo]), total, w_scale,
                                        q_scale);
        wsum += w;
        s_tile[tid] = w;
        __syncthreads();
        for (uint32_t i = 0; i < min(256u, hi - base); i++) {
            const int32_t wi = s_tile[i];
            if (!wi) continue;
            const int32_t* v = view.value(base + i);
            for (int c = 0; c < 2; c++)
                if (tid + 256 * c < hd) acc[c] += (uint64_t)((int64_t)wi * v[tid + 256 * c]);
        }
        __syncthreads();
    }
    wsum = wave_sum_sat32(wsum);
    if (lane == 0) s_w[wave] = wsum;
    __syncthreads();
    const int64_t resid = dn::ONE_ACT - (s_w[0] + s_w[1] + s_w[2] + s_w[3]);
    const int32_t* v = view.value(best.i);
    for (int c = 0; c < 2; c++)
        if (tid + 256 * c < hd)
            out[tid + 256 * c] = dn::requantize((int64_t)(acc[c] + (uint64_t)(resid * v[tid + 256 * c])));
}

// A place of zeros for keys whose page is outside the cache.
__device__ const int32_t g_zeros[ATTN_MAX_HEAD_DIM] = {};

struct TreeView {
    const int32_t *k, *v, *table;
    uint32_t pages, page_size, page_log, length, window, pos;
    size_t page_stride;
    uint32_t hd;
    uint64_t mask;
    const uint64_t* masks;  // of the request's rows
    int32_t* status;
    __device__ bool sees(uint32_t j) const {
        if (j < length) return true;
        const uint32_t i = j - length;
        if (!((mask >> i) & 1)) return false;
        return !window || pos - (length + __popcll(masks[i]) - 1) < window;
    }
    __device__ const int32_t* at(const int32_t* base, uint32_t j) const {
        const uint32_t page = (uint32_t)table[j >> page_log];
        if (page >= pages) {
            if (status) *status = IRIS_E_INVALID;
            return g_zeros;
        }
        return base + (size_t)page * page_stride + (size_t)(j & (page_size - 1)) * hd;
    }
    __device__ const int32_t* key(uint32_t j) const { return at(k, j); }
    __device__ const int32_t* value(uint32_t j) const { return at(v, j); }
};

__global__ __launch_bounds__(256) void tree_kernel(const IrisPagedKv c, const IrisTreeAttention a, int32_t* space) {
    __shared__ uint64_t s_mask[TREE_MAX_NODES];
    const uint32_t i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, g = h / (a.heads / c.kv_heads);
    const int64_t r0 = a.row_start[b], r1 = a.row_start[b + 1], len = a.lengths[b], n = r1 - r0;
    if (n <= 0) return;
    if (r0 < 0 || r1 > a.rows || n > a.max_nodes || len < 0 || len + n > a.max_positions ||
        len + n > (int64_t)a.table_stride * c.page_size) {
        if (a.status && threadIdx.x == 0) *a.status = IRIS_E_RANGE;
        return;
    }
    if (i >= n) return;
    const uint64_t mask = tree_ancestors(a.parents ? a.parents + r0 : nullptr, (uint32_t)n, threadIdx.x & 63);
    if (threadIdx.x < 64) s_mask[threadIdx.x] = mask;
    __syncthreads();
    const uint32_t pos = (uint32_t)len + __popcll(s_mask[i]) - 1;
    const uint32_t lo = a.window && pos + 1 > a.window ? min(pos + 1 - a.window, (uint32_t)len) : 0;
    const uint32_t hd = c.head_dim;
    TreeView v{c.k + (size_t)g * c.page_size * hd, c.v + (size_t)g * c.page_size * hd,
               a.table + (size_t)b * a.table_stride, c.pages, c.page_size, 31u - __clz((int)c.page_size), (uint32_t)len,
               a.window, pos, (size_t)c.kv_heads * c.page_size * hd, hd, s_mask[i], s_mask, a.status};
    const size_t row = (size_t)r0 + i;
    attend_one(v, a.q + row * a.q_stride + (size_t)h * hd, a.out + row * a.out_stride + (size_t)h * hd, lo,
               (uint32_t)(len + n), hd, a.scaled, a.scale_q32, space + (row * a.heads + h) * a.max_positions);
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

int tree_check(const IrisPagedKv* c, const IrisTreeAttention* a) {
    const int rc = iris_paged_check(c);
    if (rc) return rc;
    if (!a || !a->q || !a->out || !a->row_start || !a->lengths || !a->table) return IRIS_E_INVALID;
    if (misaligned(a->q) || misaligned(a->out) || (a->q_stride | a->out_stride) % 4) return IRIS_E_INVALID;
    if (!a->heads || a->heads % c->kv_heads || a->heads > 65535) return IRIS_E_INVALID;
    const uint64_t q = (uint64_t)a->heads * c->head_dim;
    if (a->q_stride < q || a->out_stride < q || !a->table_stride || !a->max_nodes || !a->max_positions)
        return IRIS_E_INVALID;
    if (a->max_nodes > TREE_MAX_NODES || a->max_positions > TREE_MAX_POSITIONS || a->rows > INT32_MAX ||
        a->requests > 65535)
        return IRIS_E_RANGE;
    return 0;
}

}  // namespace

extern "C" {

uint64_t iris_attention_tree_workspace_bytes(const IrisPagedKv* c, const IrisTreeAttention* a) {
    if (tree_check(c, a)) return 0;
    return (uint64_t)a->rows * a->heads * a->max_positions * 4;
}

int iris_attention_tree(const IrisPagedKv* c, const IrisTreeAttention* a, void* space, uint64_t bytes, void* stream) {
    const int rc = tree_check(c, a);
    if (rc) return rc;
    if (!a->rows || !a->requests) return 0;
    if (!space || misaligned(space)) return IRIS_E_INVALID;
    if (bytes < iris_attention_tree_workspace_bytes(c, a)) return IRIS_E_RANGE;
    hipLaunchKernelGGL(tree_kernel, dim3(a->max_nodes, a->heads, a->requests), dim3(256), 0, (hipStream_t)stream, *c, *a,
                       (int32_t*)space);
    return (int)hipGetLastError();
}

}  // extern "C"
