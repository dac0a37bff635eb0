// The paged cache of several requests: block tables and slot map of a pass
// (iris_paged_plan) and the store of its keys and values (iris_paged_store).
#include <algorithm>

#include "paged.h"

namespace {

constexpr uint32_t PLAN_MAX_REQUESTS = 4096;
constexpr uint32_t PLAN_THREADS = 1024;
// Added rows a plan workgroup takes: below two of these one workgroup does
// all of a plan. (60011 rows of 2048 requests: 29 workgroups 13 us, one 87.)
constexpr uint32_t PLAN_ROWS = 2048;

// A request's part of the plan, and the running sums before it.
struct PlanSums {
    int64_t rows, pops, pushes;
};

__device__ __forceinline__ PlanSums operator+(PlanSums a, PlanSums b) {
    return {a.rows + b.rows, a.pops + b.pops, a.pushes + b.pushes};
}

__device__ __forceinline__ PlanSums shfl_up(PlanSums v, int by) {
    return {__shfl_up(v.rows, by), __shfl_up(v.pops, by), __shfl_up(v.pushes, by)};
}

// The last of s[0 .. n] (ascending, s[0] = 0) that is at most x: the request
// of item x.
__device__ __forceinline__ uint32_t request_of(const int32_t* s, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;  // s[lo] <= x < s[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Every workgroup forms the running sums over all requests (a few values per
// thread), then takes its share of the rows, the fresh table entries and the
// returned pages. In-place launches (held_out = held, ring_state_out =
// ring_state) of several workgroups leave those two arrays to a second launch
// of one (`counts_only`), since others may not have read them yet.
//
// Bound by latency: the lengths, the sums' scan, a table entry per row, in a
// chain. 8 requests of one row 4.4 us; 2048 of 60011 rows, 29 workgroups, 13.2
// us (the rows alone are 0.5 MB).
__global__ __launch_bounds__(PLAN_THREADS) void plan_kernel(const IrisPagedPlan p, int write_counts, int counts_only) {
    extern __shared__ int32_t s_plan[];
    __shared__ PlanSums s_wave[PLAN_THREADS / 64];
    __shared__ int s_status;
    const uint32_t n = p.requests, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x;
    int32_t* s_row = s_plan;         // [n + 1] running sums
    int32_t* s_pop = s_row + n + 1;
    int32_t* s_push = s_pop + n + 1;
    int32_t* s_len = s_push + n + 1;  // [n]
    int32_t* s_held = s_len + n;
    const int32_t page_log = 31 - __clz((int)p.page_size);
    const int64_t stride = p.table_stride;
    const int32_t head = p.ring_state[0], free = p.ring_state[1];
    if (tid == 0) s_status = head < 0 || (uint32_t)head >= p.pages || free < 0 || (uint32_t)free > p.pages ? 2 : 0;
    __syncthreads();

    // Requests per thread in a row, so that the thread's sums are in order.
    const uint32_t per = (n + threads - 1) / threads, b0 = min(tid * per, n), b1 = min(b0 + per, n);
    PlanSums mine{0, 0, 0};
    int bad = 0;
    for (uint32_t b = b0; b < b1; b++) {
        const int64_t len = p.lengths[b], add = p.added[b], held = p.held[b];
        const int64_t need = (len + add + p.page_size - 1) >> page_log;
        if (len < 0 || add < 0 || held < 0 || held > stride || (held << page_log) < len) bad = IRIS_E_INVALID;
        else if (need > stride || (p.parents && add > TREE_MAX_NODES)) bad = bad ? bad : IRIS_E_RANGE;
        s_len[b] = (int32_t)len;
        s_held[b] = (int32_t)held;
        mine.rows += add;
        mine.pops += max((int64_t)0, need - held);
        mine.pushes += max((int64_t)0, held - need);
    }
    PlanSums run = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const PlanSums o = shfl_up(run, off);
        if ((int)lane >= off) run = run + o;
    }
    if (lane == 63) s_wave[wave] = run;
    // 2: counts that cannot be; 1: too many of something.
    if (bad == IRIS_E_INVALID) atomicMax(&s_status, 2);
    if (bad == IRIS_E_RANGE) atomicMax(&s_status, 1);
    __syncthreads();
    PlanSums before{run.rows - mine.rows, run.pops - mine.pops, run.pushes - mine.pushes}, total{0, 0, 0};
    for (uint32_t w = 0; w < threads / 64; w++) {
        if (w < wave) before = before + s_wave[w];
        total = total + s_wave[w];
    }
    int status = s_status == 2 ? IRIS_E_INVALID : s_status == 1 ? IRIS_E_RANGE : 0;
    if (!status && (total.rows > p.max_rows || total.pops > free)) status = IRIS_E_RANGE;
    // (More than the ring has places for: pages would go back to where others are taken.)
    if (!status && free + total.pushes > p.pages) status = IRIS_E_INVALID;
    const bool ok = status == 0;
    const bool first = blockIdx.x == 0;
    for (uint32_t b = b0; b < b1; b++) {
        s_row[b] = (int32_t)before.rows;
        s_pop[b] = (int32_t)before.pops;
        s_push[b] = (int32_t)before.pushes;
        const int64_t need = ((int64_t)s_len[b] + p.added[b] + p.page_size - 1) >> page_log;
        before.rows += p.added[b];
        before.pops += max((int64_t)0, need - s_held[b]);
        before.pushes += max((int64_t)0, s_held[b] - need);
    }
    if (tid == 0) {
        s_row[n] = (int32_t)total.rows;
        s_pop[n] = (int32_t)total.pops;
        s_push[n] = (int32_t)total.pushes;
    }
    __syncthreads();  // also: every held and ring_state of this workgroup is read
    if (write_counts && first) {
        for (uint32_t b = tid; b < n; b += threads)
            p.held_out[b] = ok ? s_held[b] + (s_pop[b + 1] - s_pop[b]) - (s_push[b + 1] - s_push[b]) : s_held[b];
        if (tid == 0) {
            p.ring_state_out[0] = ok ? (int32_t)(((int64_t)head + total.pops) % p.pages) : head;
            p.ring_state_out[1] = ok ? (int32_t)(free - total.pops + total.pushes) : free;
        }
    }
    if (counts_only) return;
    if (first) {
        for (uint32_t b = tid; b <= n; b += threads) p.row_start[b] = ok ? s_row[b] : 0;
        if (tid == 0) *p.status = status;
    }
    const uint32_t step = gridDim.x * threads, item0 = blockIdx.x * threads + tid;
    const int32_t rows = ok ? s_row[n] : 0;
    // A free page by its place in the ring.
    auto ring_page = [&](int64_t place) { return p.ring[(uint64_t)(head + place) % p.pages]; };
    for (uint32_t r = item0; r < p.max_rows; r += step) {
        int32_t slot = -1, pos = -1;
        if ((int32_t)r < rows) {
            const uint32_t b = request_of(s_row, n, (int32_t)r);
            const int32_t at = s_len[b] + (int32_t)r - s_row[b], col = at >> page_log;
            const int32_t page = col < s_held[b] ? p.table[(size_t)b * stride + col]
                                                 : ring_page((int64_t)s_pop[b] + col - s_held[b]);
            slot = page < 0 || (uint32_t)page >= p.pages ? -1 : (page << page_log) | (at & ((int32_t)p.page_size - 1));
            pos = at;
        }
        p.slots[r] = slot;
        if (p.positions && (!p.parents || pos < 0)) p.positions[r] = pos;
    }
    if (!ok) return;
    for (int32_t i = (int32_t)item0; i < s_pop[n]; i += (int32_t)step) {
        const uint32_t b = request_of(s_pop, n, i);
        p.table[(size_t)b * stride + s_held[b] + (i - s_pop[b])] = ring_page(i);
    }
    for (int32_t i = (int32_t)item0; i < s_push[n]; i += (int32_t)step) {
        const uint32_t b = request_of(s_push, n, i);
        const int32_t need = s_held[b] - (s_push[b + 1] - s_push[b]);
        p.ring[(uint64_t)((int64_t)head + free + i) % p.pages] = p.table[(size_t)b * stride + need + (i - s_push[b])];
    }
    if (!p.parents || !p.positions) return;
    // Trees: a wave per request, a lane per row.
    for (uint32_t b = blockIdx.x * (threads / 64) + wave; b < n; b += gridDim.x * (threads / 64)) {
        const uint32_t r0 = (uint32_t)s_row[b], rn = (uint32_t)s_row[b + 1] - r0;
        const uint64_t above = tree_ancestors(p.parents + r0, rn, lane);
        if (lane < rn) p.positions[r0 + lane] = s_len[b] + __popcll(above) - 1;
    }
}

// Four values of one row to their slot per thread and turn: rows of width / 4
// pieces, keys then values. Bound by memory: 6007 rows of 8 heads of 128, 98 MB
// read and written, 15.2 us where the same buffers come again and the last-level
// cache holds them (a copy of as many bytes 14.5), 18.9 us over sixteen sets in
// turn (the copy 20.4); 8 rows 2.1 us.
__global__ __launch_bounds__(256) void store_kernel(const IrisPagedKv c, const int32_t* k, uint32_t k_stride,
                                                    const int32_t* v, uint32_t v_stride, const int32_t* slots) {
    const uint32_t hd4 = c.head_dim / 4, w4 = c.kv_heads * hd4, page_log = 31 - __clz((int)c.page_size);
    const uint32_t row = blockIdx.x;
    const int32_t slot = slots[row];
    if (slot < 0 || (uint32_t)slot >= c.pages * c.page_size) return;
    const size_t page = (uint32_t)slot >> page_log, place = (uint32_t)slot & (c.page_size - 1);
    const int4* ks = (const int4*)(k + (size_t)row * k_stride);
    const int4* vs = (const int4*)(v + (size_t)row * v_stride);
    for (uint32_t i = threadIdx.x; i < w4; i += 256) {
        const uint32_t g = i / hd4, d = i % hd4;
        const size_t at = ((page * c.kv_heads + g) * c.page_size + place) * hd4 + d;
        ((int4*)c.k)[at] = ks[i];
        ((int4*)c.v)[at] = vs[i];
    }
}

}  // namespace

int iris_paged_check(const IrisPagedKv* c) {
    if (!c || !c->k || !c->v || misaligned(c->k) || misaligned(c->v)) return IRIS_E_INVALID;
    if (!c->pages || !c->kv_heads || c->kv_heads > 65535 || !c->head_dim || c->head_dim % 4 || c->head_dim > ATTN_MAX_HEAD_DIM)
        return IRIS_E_INVALID;
    if (c->page_size < 4 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return IRIS_E_INVALID;
    if ((uint64_t)c->pages * c->page_size > INT32_MAX) return IRIS_E_RANGE;
    return 0;
}

extern "C" {

int iris_paged_plan(const IrisPagedPlan* p, void* stream) {
    if (!p || !p->lengths || !p->added || !p->held || !p->held_out || !p->table || !p->ring || !p->ring_state ||
        !p->ring_state_out || !p->row_start || !p->slots || !p->status)
        return IRIS_E_INVALID;
    if (!p->requests || !p->table_stride || !p->pages) return IRIS_E_INVALID;
    if (p->page_size < 4 || p->page_size > 1024 || (p->page_size & (p->page_size - 1))) return IRIS_E_INVALID;
    if ((uint64_t)p->pages * p->page_size > INT32_MAX || (uint64_t)p->table_stride * p->page_size > INT32_MAX ||
        p->max_rows > INT32_MAX || p->requests > PLAN_MAX_REQUESTS)
        return IRIS_E_RANGE;
    const uint32_t groups = std::max(1u, std::min(p->max_rows / PLAN_ROWS, 128u));
    // Four waves scan few requests sooner than sixteen: 8 requests 4.4 / 6.3 us.
    const uint32_t threads = p->requests <= 256 && groups == 1 && p->max_rows <= 1024 ? 256 : PLAN_THREADS;
    const size_t lds = (5 * (size_t)p->requests + 3) * 4;
    const bool in_place = p->held_out == p->held || p->ring_state_out == p->ring_state;
    const int split = in_place && groups > 1;
    const hipError_t st = paged_lds_limit((const void*)plan_kernel, lds);
    if (st != hipSuccess) return (int)st;
    hipLaunchKernelGGL(plan_kernel, dim3(groups), dim3(threads), lds, (hipStream_t)stream, *p, !split, 0);
    if (split) hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(threads), lds, (hipStream_t)stream, *p, 1, 1);
    return (int)hipGetLastError();
}

int iris_paged_store(const IrisPagedKv* c, const int32_t* k, uint32_t k_stride, const int32_t* v, uint32_t v_stride,
                     const int32_t* slots, uint32_t rows, void* stream) {
    const int rc = iris_paged_check(c);
    if (rc) return rc;
    const uint64_t width = (uint64_t)c->kv_heads * c->head_dim;
    if (!k || !v || !slots || misaligned(k) || misaligned(v) || k_stride % 4 || v_stride % 4 || k_stride < width ||
        v_stride < width)
        return IRIS_E_INVALID;
    if (rows >= 1u << 24) return IRIS_E_RANGE;  // a launch has under 2^32 threads
    if (!rows) return 0;
    hipLaunchKernelGGL(store_kernel, dim3(rows), dim3(256), 0, (hipStream_t)stream, *c, k, k_stride, v, v_stride, slots);
    return (int)hipGetLastError();
}

}  // extern "C"
