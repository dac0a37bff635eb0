// Greedy generation of several requests at a time over one paged cache: the
// prompts of a pass packed row after row, then passes in which each request
// adds its last token, alone or with a tree of drafted continuations.
//
// A pass is a session's, layer by layer (iris_session_pass), over the rows of
// all its requests; only what lies between a layer's q|k|v product and its O
// product is the batch's own (iris_batch_attention). The pass's block tables,
// slots and positions come from iris_paged_plan, each layer's keys and values
// go to their pages with iris_paged_store; prompts attend with
// iris_attention_packed, newest rows with iris_attention_tree. Rows do not
// depend on the rows beside them, so a request's tokens are those that
// iris_session_generate selects (executor.rs:143-185).
//
// Of a tree, the rows on the path of the model's own choices are kept: from
// the root, the child whose token is the row's selection, and so on. Kept rows
// need not lie one after the other in the cache; batch_keep_kernel moves their
// keys and values to the positions behind the request's last.
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

#include "detnum_dev.h"
#include "paged.h"
#include "runtime_internal.h"

#define RT_CHECK(expr)                  \
    do {                                \
        int rc_ = (int)(expr);          \
        if (rc_ != 0) return rc_;       \
    } while (0)

namespace {

constexpr uint32_t SELECT_PARTS = 64;  // pieces of a row's logits, a workgroup each
constexpr uint32_t LOGITS_ROWS = 64;   // rows whose logits are held at a time

// Queries and keys of the q|k|v rows, rotated in place (mistral.rs:114-126):
// pair j of a head by its position's angle j.
__global__ __launch_bounds__(256) void batch_rotate_kernel(int32_t* qkv, uint32_t stride, uint32_t width, uint32_t head_dim,
                                                           const int64_t* rope_sc, const int32_t* positions) {
    const uint32_t row = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= width / 2 || positions[row] == 0) return;
    const uint32_t half = head_dim / 2, j = i % half;
    int32_t* x = qkv + (size_t)row * stride + 2 * i;
    const int64_t* sc = rope_sc + ((size_t)row * half + j) * 2;
    int32_t x0 = x[0], x1 = x[1];
    dn::rotate_pair_sc(x0, x1, sc[0], sc[1]);
    x[0] = x0;
    x[1] = x1;
}

// out[i] = the row x[at[i]] (hidden values, a multiple of 32).
__global__ __launch_bounds__(256) void batch_gather_kernel(const int32_t* x, const int32_t* at, uint32_t hidden, int32_t* out) {
    const int4* from = (const int4*)(x + (size_t)at[blockIdx.x] * hidden);
    int4* to = (int4*)(out + (size_t)blockIdx.x * hidden);
    for (uint32_t i = threadIdx.x; i < hidden / 4; i += 256) to[i] = from[i];
}

// A logit and its index as one key: larger for a larger logit, of equal ones
// for the smaller index.
__device__ __forceinline__ int64_t select_key(int32_t v, uint32_t i) { return (int64_t)v << 32 | (uint32_t)~i; }

__device__ __forceinline__ int64_t wave_max(int64_t k) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) k = max(k, (int64_t)__shfl_xor((long long)k, off));
    return k;
}

// The first maximum of each piece of a row's logits.
__global__ __launch_bounds__(256) void batch_select_kernel(const int32_t* logits, uint32_t vocab, int64_t* best) {
    __shared__ int64_t s_best[4];
    const uint32_t per = (vocab + SELECT_PARTS - 1) / SELECT_PARTS;
    const uint32_t i0 = blockIdx.x * per, i1 = min(i0 + per, vocab);
    const int32_t* row = logits + (size_t)blockIdx.y * vocab;
    int64_t k = INT64_MIN;
    for (uint32_t i = i0 + threadIdx.x; i < i1; i += 256) k = max(k, select_key(row[i], i));
    k = wave_max(k);
    if (threadIdx.x % 64 == 0) s_best[threadIdx.x / 64] = k;
    __syncthreads();
    if (threadIdx.x == 0)
        best[(size_t)blockIdx.y * SELECT_PARTS + blockIdx.x] = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
}

// Each prompt's next token: the first maximum over its last row's pieces.
__global__ __launch_bounds__(64) void batch_token_kernel(const int64_t* best, int32_t* tokens) {
    static_assert(SELECT_PARTS == 64, "a lane each");
    const int64_t k = wave_max(best[(size_t)blockIdx.x * SELECT_PARTS + threadIdx.x]);
    if (threadIdx.x == 0) tokens[blockIdx.x] = (int32_t)~(uint32_t)k;
}

// One request's tree, a lane per row: each row's selection, and from the root
// (row 0) the path of rows whose token is their parent's selection (of equal
// children the first). tokens: the selections along the path, path: its rows;
// kept: their number.
__global__ __launch_bounds__(64) void batch_accept_kernel(const int64_t* best, const int32_t* row_start, const int32_t* ids,
                                                          const int32_t* parents, int32_t* tokens, int32_t* path,
                                                          int32_t* kept) {
    const uint32_t b = blockIdx.x, lane = threadIdx.x, at = row_start[b], n = row_start[b + 1] - at;
    int64_t k = INT64_MIN;
    int32_t id = -1, parent = -1;
    if (lane < n) {
        const int64_t* row = best + (size_t)(at + lane) * SELECT_PARTS;
        for (uint32_t i = 0; i < SELECT_PARTS; i++) k = max(k, row[i]);
        id = ids[at + lane];
        parent = parents ? parents[at + lane] : (int32_t)lane - 1;
    }
    const int32_t token = (int32_t)~(uint32_t)k;
    uint32_t row = 0, count = 0;
    while (count < n) {  // a path has at most n rows: each lies behind its parent
        const int32_t next = __shfl(token, row);
        if (lane == 0) tokens[at + count] = next, path[at + count] = (int32_t)row;
        count++;
        const uint64_t child = __ballot(lane < n && lane > row && parent == (int32_t)row && id == next);
        if (!child) break;
        row = __builtin_ctzll(child);
    }
    if (lane == 0) kept[b] = (int32_t)count;
}

// The keys and values of a layer's kept rows, moved to the slots behind the
// request's last. A kept row lies at or behind the slot it moves to, and a
// thread moves its part of all of them in order, so that none is overwritten
// before it is read.
__global__ __launch_bounds__(256) void batch_keep_kernel(const IrisPagedKv* caches, const int32_t* row_start,
                                                         const int32_t* path, const int32_t* kept, const int32_t* slots) {
    const IrisPagedKv c = caches[blockIdx.y];
    if (!c.k) return;  // the layer reads another's
    const uint32_t b = blockIdx.x, at = row_start[b], n = kept[b];
    uint32_t first = 1;  // the first row that moves
    while (first < n && path[at + first] == (int32_t)first) first++;
    if (first >= n) return;
    const uint32_t q = c.head_dim / 4;
    auto place = [&](int32_t slot, uint32_t i) {  // of the value i (of four) of a slot's row
        const uint32_t page = (uint32_t)slot / c.page_size, in = (uint32_t)slot % c.page_size;
        return (((size_t)page * c.kv_heads + i / q) * c.page_size + in) * q + i % q;
    };
    for (uint32_t i = threadIdx.x; i < c.kv_heads * q; i += 256)
        for (uint32_t j = first; j < n; j++) {
            const size_t from = place(slots[at + path[at + j]], i), to = place(slots[at + j], i);
            const int4 k = ((const int4*)c.k)[from], v = ((const int4*)c.v)[from];
            ((int4*)c.k)[to] = k;
            ((int4*)c.v)[to] = v;
        }
}

}  // namespace

struct IrisBatch {
    IrisSession* s = nullptr;
    uint32_t requests = 0, pages = 0, page_size = 0, table_stride = 0, max_positions = 0;
    std::vector<uint32_t> length, held;  // per request, as the device's
    bool broken = false;                 // a pass failed on the device: its state is unknown
    std::vector<IrisPagedKv> caches;     // per layer; k null: the layer reads another's
    IrisPagedKv* d_caches = nullptr;
    std::vector<int32_t*> k_rows, v_rows;  // gemma-dense: per layer, the pass's keys and values
    // What a pass brings: lengths, added, ids, parents, rows to select from.
    int32_t *host_in = nullptr, *in = nullptr;
    // What it takes back: status, kept, tokens.
    int32_t *host_out = nullptr, *out = nullptr;
    int32_t *d_held = nullptr, *table = nullptr, *ring = nullptr, *ring_state = nullptr, *row_start = nullptr;
    int32_t *slots = nullptr, *path = nullptr, *logits = nullptr;
    int64_t* best = nullptr;
    void* space = nullptr;  // of the attention
    uint64_t space_bytes = 0, space_most = 0;  // now; that a pass can need
    // The pass at hand: its requests' rows and, of prompts, the longest; of
    // newest rows, the most of a request and the last position's end.
    bool prompts = false, trees = false;
    uint32_t longest = 0, end = 0;

    int32_t* lengths() const { return in; }
    int32_t* added() const { return in + requests; }
    int32_t* picks() const { return in + 2 * requests; }
    int32_t* ids() const { return in + 3 * requests; }
    int32_t* parents() const { return in + 3 * requests + s->max_rows; }
    int32_t* status() const { return out; }
    int32_t* kept() const { return out + 1; }
    int32_t* tokens() const { return out + 1 + requests; }
    size_t in_ints() const { return 3 * (size_t)requests + 2 * (size_t)s->max_rows; }
    size_t out_ints() const { return 1 + (size_t)requests + std::max(s->max_rows, requests); }
};

// The operators' arguments for layer l of the pass at hand.
static IrisPackedAttention batch_prompts(const IrisBatch* b, uint32_t l, uint32_t rows) {
    const IrisSession* s = b->s;
    const IrisModelDesc& d = s->model->d;
    const LayerWeights& L = s->model->layers[l];
    const bool gemma = d.family == IRIS_FAMILY_GEMMA_DENSE;
    const uint32_t qw = L.q_rows, kvw = L.kv_rows, qkvw = qw + 2 * kvw;
    IrisPackedAttention a{};
    a.q = gemma ? s->q : s->qkv;
    a.k = gemma ? b->k_rows[L.kv_source] : s->qkv + qw;
    a.v = gemma ? b->v_rows[L.kv_source] : s->qkv + qw + kvw;
    a.out = s->ctx;
    a.row_start = b->row_start;
    a.q_stride = gemma ? qw : qkvw, a.k_stride = a.v_stride = gemma ? kvw : qkvw, a.out_stride = qw;
    a.sequences = b->requests, a.rows = rows, a.max_length = b->longest;
    a.heads = d.heads, a.kv_heads = d.kv_heads, a.head_dim = L.head_dim, a.window = L.window;
    a.scaled = !gemma, a.scale_q32 = gemma ? 0 : d.attention_scale_q32;
    return a;
}

static IrisTreeAttention batch_newest(const IrisBatch* b, uint32_t l, uint32_t rows) {
    const IrisSession* s = b->s;
    const IrisModelDesc& d = s->model->d;
    const LayerWeights& L = s->model->layers[l];
    const bool gemma = d.family == IRIS_FAMILY_GEMMA_DENSE;
    IrisTreeAttention a{};
    a.q = gemma ? s->q : s->qkv, a.out = s->ctx;
    a.row_start = b->row_start, a.lengths = b->lengths(), a.parents = b->trees ? b->parents() : nullptr, a.table = b->table;
    a.q_stride = gemma ? L.q_rows : L.q_rows + 2 * L.kv_rows, a.out_stride = L.q_rows;
    a.requests = b->requests, a.rows = rows, a.table_stride = b->table_stride;
    a.max_nodes = b->longest, a.max_positions = b->end;
    a.heads = d.heads, a.window = L.window;
    a.scaled = !gemma, a.scale_q32 = gemma ? 0 : d.attention_scale_q32;
    return a;
}

// Work space for the pass at hand, before it begins: where the device has
// none, the pass is refused (hipErrorOutOfMemory) and the requests stay as they
// were. It grows by halves up to what the largest pass takes, since positions
// grow from pass to pass and each growth waits for the device.
static int batch_space(IrisBatch* b, uint32_t rows) {
    uint64_t need = 0;
    for (uint32_t l = 0; rows && l < b->s->model->d.layers; l++) {
        if (b->prompts) {
            const IrisPackedAttention a = batch_prompts(b, l, rows);
            need = std::max(need, iris_attention_packed_workspace_bytes(&a));
        } else {
            const IrisTreeAttention a = batch_newest(b, l, rows);
            need = std::max(need, iris_attention_tree_workspace_bytes(&b->caches[b->s->model->layers[l].kv_source], &a));
        }
    }
    if (need <= b->space_bytes) return 0;
    uint64_t bytes = std::max(need, std::min(b->space_bytes + b->space_bytes / 2, b->space_most));
    RT_CHECK(hipStreamSynchronize(b->s->stream));
    (void)hipFree(b->space);
    b->space = nullptr;
    b->space_bytes = 0;
    hipError_t st = hipMalloc(&b->space, bytes);
    if (st != hipSuccess && bytes > need) st = hipMalloc(&b->space, bytes = need);
    if (st != hipSuccess) {
        b->space = nullptr;
        (void)hipGetLastError();  // returned here: not the next launch's to report
        return (int)st;
    }
    b->space_bytes = bytes;
    return 0;
}

int iris_batch_attention(IrisSession* s, uint32_t l, uint32_t rows) {
    IrisBatch* b = s->batch;
    const IrisModel* m = s->model;
    const IrisModelDesc& d = m->d;
    const LayerWeights& L = m->layers[l];
    const bool gemma = d.family == IRIS_FAMILY_GEMMA_DENSE, own = L.kv_source == (int32_t)l;
    const uint32_t hd = L.head_dim, qw = L.q_rows, kvw = L.kv_rows, qkvw = qw + 2 * kvw;
    hipStream_t st = s->stream;
    if (gemma) {
        GemmaQkvArgs qa{};
        qa.qkv = s->qkv;
        qa.qkv_stride = qkvw;
        qa.heads = d.heads;
        qa.kv_heads = d.kv_heads;
        qa.head_dim = hd;
        qa.rotary_dim = L.rotary_dim;
        qa.q_norm = L.q_norm;
        qa.k_norm = L.k_norm;
        qa.eps = d.norm_eps;
        qa.inv_freq = L.inv_freq;
        qa.positions = s->d_pos;
        qa.q_out = s->q;
        qa.q_stride = qw;
        if (own) qa.k_rows = b->k_rows[l], qa.v_rows = b->v_rows[l];
        RT_CHECK(iris_gemma_qkv_finish_launch(qa, rows, st));
    } else {
        hipLaunchKernelGGL(batch_rotate_kernel, dim3(((qw + kvw) / 2 + 255) / 256, rows), dim3(256), 0, st, s->qkv, qkvw, qw + kvw,
                           hd, s->rope_sc, s->d_pos);
        RT_CHECK(hipGetLastError());
    }
    // The layer's queries, and the keys and values its attention reads.
    const IrisPackedAttention prompts = batch_prompts(b, l, rows);
    const IrisPagedKv& cache = b->caches[L.kv_source];
    if (own) RT_CHECK(iris_paged_store(&cache, prompts.k, prompts.k_stride, prompts.v, prompts.v_stride, b->slots, rows, st));
    if (b->prompts) return iris_attention_packed(&prompts, b->space, b->space_bytes, st);
    const IrisTreeAttention newest = batch_newest(b, l, rows);
    return iris_attention_tree(&cache, &newest, b->space, b->space_bytes, st);
}

// First maxima of the logits of `count` rows of x, as SELECT_PARTS keys each.
static int batch_select(IrisBatch* b, const int32_t* x, uint32_t count) {
    IrisSession* s = b->s;
    const IrisModel* m = s->model;
    const uint32_t H = m->d.hidden, V = m->d.vocab;
    for (uint32_t r = 0; r < count; r += LOGITS_ROWS) {
        const uint32_t n = std::min(LOGITS_ROWS, count - r);
        GemvArgs g{};
        g.w = q8_view(m->head);
        g.x = x + (size_t)r * H;
        g.x_stride = H;
        g.tokens = n;
        g.prologue = PRO_RMSNORM;
        g.norm_w = m->final_norm;
        g.norm_eps = m->d.norm_eps;
        g.epilogue = EPI_SOFTCAP;
        g.softcap = m->head_softcap;
        g.out = b->logits;
        g.out_stride = V;
        if (n > 1) {
            g.planes = s->planes;
            g.token_limbs = s->token_limbs;
        }
        RT_CHECK(iris_gemv_launch(g, s->stream));
        hipLaunchKernelGGL(batch_select_kernel, dim3(SELECT_PARTS, n), dim3(256), 0, s->stream, b->logits, V,
                           b->best + (size_t)r * SELECT_PARTS);
        RT_CHECK(hipGetLastError());
    }
    return 0;
}

// One pass over the requests' rows that host_in holds.
static int batch_pass(IrisBatch* b, uint32_t rows, uint32_t picks) {
    IrisSession* s = b->s;
    const IrisModel* m = s->model;
    hipStream_t st = s->stream;
    RT_CHECK(hipMemcpyAsync(b->in, b->host_in, b->in_ints() * 4, hipMemcpyHostToDevice, st));
    IrisPagedPlan p{};
    p.lengths = b->lengths(), p.added = b->added(), p.parents = b->trees ? b->parents() : nullptr;
    p.held = p.held_out = b->d_held;
    p.table = b->table, p.ring = b->ring, p.ring_state = p.ring_state_out = b->ring_state;
    p.row_start = b->row_start, p.slots = b->slots, p.positions = s->d_pos, p.status = b->status();
    p.requests = b->requests, p.table_stride = b->table_stride, p.pages = b->pages, p.page_size = b->page_size;
    p.max_rows = std::max(rows, 1u);
    RT_CHECK(iris_paged_plan(&p, st));
    if (rows) {
        RT_CHECK(hipMemcpyAsync(s->ids, b->ids(), (size_t)rows * 4, hipMemcpyDeviceToDevice, st));
        RT_CHECK(iris_embed_rows_launch(s->ids, rows, m->embed_raw, m->embed_row_bytes, m->d.hidden, m->embed_scale, s->x, st));
        s->rope_ready = false;
        RT_CHECK(iris_session_pass(s, rows, nullptr));
        if (b->prompts) {
            hipLaunchKernelGGL(batch_gather_kernel, dim3(picks), dim3(256), 0, st, s->x, b->picks(), m->d.hidden, s->attended);
            RT_CHECK(hipGetLastError());
            RT_CHECK(batch_select(b, s->attended, picks));
            hipLaunchKernelGGL(batch_token_kernel, dim3(picks), dim3(64), 0, st, b->best, b->tokens());
        } else {
            RT_CHECK(batch_select(b, s->x, rows));
            hipLaunchKernelGGL(batch_accept_kernel, dim3(b->requests), dim3(64), 0, st, b->best, b->row_start, s->ids,
                               p.parents, b->tokens(), b->path, b->kept());
            RT_CHECK(hipGetLastError());
            if (b->longest > 2 && b->trees && m->d.layers)
                hipLaunchKernelGGL(batch_keep_kernel, dim3(b->requests, m->d.layers), dim3(256), 0, st, b->d_caches, b->row_start,
                                   b->path, b->kept(), b->slots);
        }
        RT_CHECK(hipGetLastError());
    }
    RT_CHECK(hipMemcpyAsync(b->host_out, b->out, b->out_ints() * 4, hipMemcpyDeviceToHost, st));
    RT_CHECK(hipStreamSynchronize(st));
    return b->host_out[0];
}

static uint32_t pages_of(const IrisBatch* b, uint64_t positions) {
    return (uint32_t)((positions + b->page_size - 1) / b->page_size);
}

// The checks of a pass, its inputs into host_in and the pass itself.
static int batch_run(IrisBatch* b, const int32_t* ids, const int32_t* parents, const uint32_t* counts, bool prompts) {
    if (b->broken) return IRIS_E_STATE;
    IrisSession* s = b->s;
    const IrisModel* m = s->model;
    const uint32_t n = b->requests;
    uint64_t rows = 0, pages = 0, held = 0, grow = 0, most = 0, end = 0;
    for (uint32_t i = 0; i < n; i++) {
        const uint64_t c = counts[i], to = b->length[i] + c;
        if (c && prompts != (b->length[i] == 0)) return IRIS_E_STATE;
        if (c && (to > b->max_positions || to > m->d.max_positions)) return IRIS_E_RANGE;
        if (c > (prompts ? ATTN_MAX_KEYS : TREE_MAX_NODES)) return IRIS_E_RANGE;
        rows += c;
        most = std::max(most, c);
        if (c) end = std::max(end, to);
        const uint32_t need = pages_of(b, to);
        pages += need;
        held += b->held[i];
        grow += need > b->held[i] ? need - b->held[i] : 0;
    }
    if (rows > s->max_rows || pages > b->pages) return IRIS_E_RANGE;
    if (rows && !ids) return IRIS_E_INVALID;
    for (uint64_t r = 0; r < rows; r++) {
        if (ids[r] < 0 || (uint32_t)ids[r] >= m->d.vocab) return IRIS_E_INVALID;
        if (iris_embedding_refused(m, ids[r])) return IRIS_E_SCALE;
    }
    int32_t* in = b->host_in;
    uint32_t picks = 0, at = 0;
    for (uint32_t i = 0; i < n; i++) {
        in[i] = (int32_t)b->length[i];
        in[n + i] = (int32_t)counts[i];
        at += counts[i];
        if (prompts && counts[i]) in[2 * n + picks++] = (int32_t)at - 1;
    }
    if (rows) std::memcpy(in + 3 * n, ids, rows * 4);
    if (rows && parents) std::memcpy(in + 3 * n + s->max_rows, parents, rows * 4);
    b->prompts = prompts;
    b->trees = parents != nullptr;
    b->longest = (uint32_t)most;
    b->end = (uint32_t)end;
    RT_CHECK(batch_space(b, (uint32_t)rows));
    b->broken = true;  // until the pass has ended well
    if (grow > b->pages - held) {
        // The plan takes pages before it gives others back, so those of
        // released requests and of rows not kept go back first.
        std::memset(in + n, 0, n * 4);
        RT_CHECK(batch_pass(b, 0, 0));
        for (uint32_t i = 0; i < n; i++) in[n + i] = (int32_t)counts[i];
    }
    RT_CHECK(batch_pass(b, (uint32_t)rows, picks));
    for (uint32_t i = 0; i < n; i++) b->held[i] = pages_of(b, b->length[i] + counts[i]);
    b->broken = false;
    return 0;
}

extern "C" {

int iris_batch_create(IrisModel* m, uint32_t requests, uint32_t pages, uint32_t page_size, uint32_t max_positions,
                      uint32_t max_rows, IrisBatch** out) {
    if (!m || !out || !m->finalized || !requests || !pages || !max_positions || !max_rows) return IRIS_E_INVALID;
    *out = nullptr;
    const IrisModelDesc& d = m->d;
    // Rows are a launch's second dimension in the layers' kernels.
    if (requests > 4096 || max_rows > 65535 || max_positions > TREE_MAX_POSITIONS)
        return IRIS_E_RANGE;
    // What the paged operators take, layer by layer (the addresses stand for
    // the pass's; nothing is read).
    int32_t* some = (int32_t*)256;
    uint64_t most = 0;
    IrisPagedKv shape{some, some, pages, page_size, 1, 4};
    RT_CHECK(iris_paged_check(&shape));
    for (const LayerWeights& L : m->layers) {
        shape.kv_heads = d.kv_heads, shape.head_dim = L.head_dim;
        RT_CHECK(iris_paged_check(&shape));
        const uint32_t stride = L.q_rows + 2 * L.kv_rows;
        IrisPackedAttention pa{};
        pa.q = pa.k = pa.v = some, pa.out = some, pa.row_start = some;
        pa.q_stride = pa.k_stride = pa.v_stride = pa.out_stride = stride;
        pa.sequences = requests, pa.rows = max_rows, pa.max_length = std::min(std::min(max_rows, max_positions), ATTN_MAX_KEYS);
        pa.heads = d.heads, pa.kv_heads = d.kv_heads, pa.head_dim = L.head_dim, pa.window = L.window;
        IrisTreeAttention ta{};
        ta.q = some, ta.out = some, ta.row_start = ta.lengths = ta.table = some;
        ta.q_stride = ta.out_stride = stride;
        ta.requests = requests, ta.rows = max_rows, ta.table_stride = (max_positions + page_size - 1) / page_size;
        ta.max_nodes = std::min(max_rows, TREE_MAX_NODES), ta.max_positions = max_positions;
        ta.heads = d.heads, ta.window = L.window;
        const uint64_t of_prompts = iris_attention_packed_workspace_bytes(&pa), of_newest = iris_attention_tree_workspace_bytes(&shape, &ta);
        if (!of_prompts || !of_newest) return IRIS_E_RANGE;
        most = std::max(most, std::max(of_prompts, of_newest));
    }
    IrisBatch* b = new (std::nothrow) IrisBatch();
    if (!b) return IRIS_E_NOMEM;
    b->space_most = most;
    b->requests = requests, b->pages = pages, b->page_size = page_size, b->max_positions = max_positions;
    b->table_stride = (max_positions + page_size - 1) / page_size;
    int rc = 0;
    try {
        b->length.assign(requests, 0);
        b->held.assign(requests, 0);
        b->caches.assign(d.layers, IrisPagedKv{});
        b->k_rows.assign(d.layers, nullptr);
        b->v_rows.assign(d.layers, nullptr);
        rc = iris_session_make(m, max_positions, max_rows, b, &b->s);
    } catch (const std::bad_alloc&) {
        rc = IRIS_E_NOMEM;
    }
    if (rc) {
        iris_batch_free(b);
        return rc;
    }
    hipError_t st = hipSuccess;
    auto alloc = [&](auto** p, uint64_t count) {
        if (st == hipSuccess) st = hipMalloc((void**)p, std::max<uint64_t>(count, 4) * sizeof(**p));
    };
    for (uint32_t l = 0; l < d.layers; l++) {
        const LayerWeights& L = m->layers[l];
        if (L.kv_source != (int32_t)l) continue;
        IrisPagedKv& c = b->caches[l];
        c.pages = pages, c.page_size = page_size, c.kv_heads = d.kv_heads, c.head_dim = L.head_dim;
        alloc(&c.k, (uint64_t)pages * page_size * L.kv_rows);
        alloc(&c.v, (uint64_t)pages * page_size * L.kv_rows);
        if (d.family == IRIS_FAMILY_GEMMA_DENSE) {
            alloc(&b->k_rows[l], (uint64_t)max_rows * L.kv_rows);
            alloc(&b->v_rows[l], (uint64_t)max_rows * L.kv_rows);
        }
    }
    alloc(&b->d_caches, d.layers);
    alloc(&b->in, b->in_ints());
    alloc(&b->out, b->out_ints());
    alloc(&b->d_held, requests);
    alloc(&b->table, (uint64_t)requests * b->table_stride);
    alloc(&b->ring, pages);
    alloc(&b->ring_state, 2);
    alloc(&b->row_start, requests + 1);
    alloc(&b->slots, max_rows);
    alloc(&b->path, max_rows);
    alloc(&b->logits, (uint64_t)std::min(LOGITS_ROWS, std::max(max_rows, requests)) * d.vocab);
    alloc(&b->best, (uint64_t)max_rows * SELECT_PARTS);
    if (st == hipSuccess) st = hipHostMalloc((void**)&b->host_in, b->in_ints() * 4);
    if (st == hipSuccess) st = hipHostMalloc((void**)&b->host_out, b->out_ints() * 4);
    if (st == hipSuccess) {
        std::memset(b->host_in, 0, b->in_ints() * 4);
        st = hipMemset(b->out, 0, b->out_ints() * 4);
    }
    if (st == hipSuccess && d.layers)
        st = hipMemcpy(b->d_caches, b->caches.data(), d.layers * sizeof(IrisPagedKv), hipMemcpyHostToDevice);
    if (st == hipSuccess) st = hipMemset(b->d_held, 0, requests * 4);
    try {
        std::vector<int32_t> ring(pages);
        for (uint32_t i = 0; i < pages; i++) ring[i] = (int32_t)i;
        const int32_t state[2] = {0, (int32_t)pages};
        if (st == hipSuccess) st = hipMemcpy(b->ring, ring.data(), (size_t)pages * 4, hipMemcpyHostToDevice);
        if (st == hipSuccess) st = hipMemcpy(b->ring_state, state, 8, hipMemcpyHostToDevice);
    } catch (const std::bad_alloc&) {
        iris_batch_free(b);
        return IRIS_E_NOMEM;
    }
    if (st == hipSuccess && max_rows > 1) st = (hipError_t)iris_q8_prepare_fold(m->head, b->s->stream);
    if (st == hipSuccess) st = hipDeviceSynchronize();
    if (st != hipSuccess) {
        iris_batch_free(b);
        (void)hipGetLastError();  // returned here: not the next launch's to report
        return (int)st;
    }
    *out = b;
    return 0;
}

void iris_batch_free(IrisBatch* b) {
    if (!b) return;
    if (b->s && b->s->stream) (void)hipStreamSynchronize(b->s->stream);
    for (auto& c : b->caches) (void)hipFree(c.k), (void)hipFree(c.v);
    for (auto p : b->k_rows) (void)hipFree(p);
    for (auto p : b->v_rows) (void)hipFree(p);
    (void)hipFree(b->d_caches);
    for (int32_t* p : {b->in, b->out, b->d_held, b->table, b->ring, b->ring_state, b->row_start, b->slots, b->path, b->logits})
        (void)hipFree(p);
    (void)hipFree(b->best);
    (void)hipFree(b->space);
    if (b->host_in) (void)hipHostFree(b->host_in);
    if (b->host_out) (void)hipHostFree(b->host_out);
    iris_session_free(b->s);
    delete b;
}

int iris_batch_prefill(IrisBatch* b, const int32_t* ids, const uint32_t* counts, int32_t* out_tokens) {
    if (!b || !counts || !out_tokens) return IRIS_E_INVALID;
    RT_CHECK(batch_run(b, ids, nullptr, counts, true));
    const int32_t* tokens = b->host_out + 1 + b->requests;
    for (uint32_t i = 0, at = 0; i < b->requests; i++) {
        out_tokens[i] = counts[i] ? tokens[at++] : -1;
        b->length[i] += counts[i];
    }
    return 0;
}

int iris_batch_step(IrisBatch* b, const int32_t* ids, const int32_t* parents, const uint32_t* counts, int32_t* out_tokens,
                    uint32_t* out_kept) {
    if (!b || !counts || !out_tokens || !out_kept) return IRIS_E_INVALID;
    RT_CHECK(batch_run(b, ids, parents, counts, false));
    const int32_t *kept = b->host_out + 1, *tokens = kept + b->requests;
    for (uint32_t i = 0, at = 0; i < b->requests; at += counts[i++]) {
        out_kept[i] = counts[i] ? (uint32_t)kept[i] : 0;
        for (uint32_t j = 0; j < counts[i]; j++) out_tokens[at + j] = j < out_kept[i] ? tokens[at + j] : -1;
        b->length[i] += out_kept[i];
    }
    return 0;
}

int iris_batch_release(IrisBatch* b, uint32_t request) {
    if (!b || request >= b->requests) return IRIS_E_INVALID;
    if (b->broken) return IRIS_E_STATE;
    b->length[request] = 0;  // its pages go back to the ring with the next pass's plan
    return 0;
}

int iris_batch_length(const IrisBatch* b, uint32_t request, uint32_t* out) {
    if (!b || !out || request >= b->requests) return IRIS_E_INVALID;
    *out = b->length[request];
    return 0;
}

}  // extern "C"
