// Low-rank adapters of many requests beside one product: row r, of adapter s,
// gets out = y + B_s (A_s x), both products exact over 16-bit weights and
// rounded once each.
//
// Two launches, since every output needs the whole of A x: t = A x for each
// row into the work space, then B t added to y.
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

#include "attn_tiles.h"
#include "q8_internal.h"

namespace {

// One part of one slot; rank 0: empty.
struct AdapterEntry {
    const int16_t* a;  // [rank][cols]
    const int16_t* b;  // [rows][stride_of(rank)]
    uint32_t rank, a_bits, b_bits, pad;
};

// B's rows are padded with zeros to whole 16-byte pieces.
__host__ __device__ __forceinline__ uint32_t stride_of(uint32_t rank) { return (rank + 7) & ~7u; }

struct AdapterShape {
    uint32_t cols, part_count, slots, max_rank;
    IrisAdapterPart parts[IRIS_ADAPTER_PARTS];
};

// A sum of products as the Q16.16 value it stands for.
__device__ __forceinline__ int32_t rounded(int64_t sum, uint32_t bits) {
    return dn::clamp_i64_to_i32(dn::rshift_rte(sum, bits));
}

// The slot of a row; -1 for none and for one outside the bank.
__device__ __forceinline__ int32_t slot_of(const IrisAdapterRows& a, uint32_t slots, uint32_t row, bool report) {
    const int32_t s = a.slots[row];
    if (s >= -1 && s < (int32_t)slots) return s;
    if (report && a.status) *a.status = IRIS_E_INVALID;
    return -1;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor((long long)v, off);
    return v;
}

// One value of t a workgroup: row blockIdx.y, value blockIdx.x of the parts'
// max_rank each.
__global__ __launch_bounds__(256) void shrink_row_kernel(const IrisAdapterRows a, const AdapterShape sh,
                                                         const AdapterEntry* table, int32_t* t) {
    __shared__ int64_t s_sum[4];
    const uint32_t row = blockIdx.y, part = blockIdx.x / sh.max_rank, j = blockIdx.x % sh.max_rank;
    const int32_t slot = slot_of(a, sh.slots, row, blockIdx.x == 0 && threadIdx.x == 0);
    if (slot < 0) return;
    const AdapterEntry e = table[slot * sh.part_count + part];
    if (j >= e.rank) return;
    const int4* x = (const int4*)(a.x + (size_t)row * a.x_stride);
    const int4* w = (const int4*)(e.a + (size_t)j * sh.cols);
    int64_t sum = 0;
    for (uint32_t i = threadIdx.x; i < sh.cols / 8; i += 256) {
        const int4 p = w[i], x0 = x[2 * i], x1 = x[2 * i + 1];
        const int32_t q[4] = {p.x, p.y, p.z, p.w}, v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            sum += (int64_t)(int16_t)q[c] * v[2 * c];
            sum += (int64_t)(q[c] >> 16) * v[2 * c + 1];
        }
    }
    sum = wave_sum(sum);
    if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        t[((size_t)row * sh.part_count + part) * sh.max_rank + j] = rounded(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], e.a_bits);
}

// One output a thread: row blockIdx.y, part blockIdx.z.
__global__ __launch_bounds__(256) void expand_row_kernel(const IrisAdapterRows a, const AdapterShape sh,
                                                         const AdapterEntry* table, const int32_t* t) {
    const uint32_t row = blockIdx.y, part = blockIdx.z, i = blockIdx.x * 256 + threadIdx.x;
    const IrisAdapterPart p = sh.parts[part];
    if (i >= p.rows) return;
    const size_t column = p.first + (size_t)i * p.step;
    const int32_t slot = slot_of(a, sh.slots, row, false);
    AdapterEntry e{};
    if (slot >= 0) e = table[slot * sh.part_count + part];
    if (!e.rank && a.out == a.y) return;
    int32_t v = a.y[(size_t)row * a.y_stride + column];
    if (e.rank) {
        const int32_t* tr = t + ((size_t)row * sh.part_count + part) * sh.max_rank;
        const int16_t* w = e.b + (size_t)i * stride_of(e.rank);
        int64_t sum = 0;
        for (uint32_t j = 0; j < e.rank; j++) sum += (int64_t)w[j] * tr[j];
        v = dn::add_sat(v, rounded(sum, e.b_bits));
    }
    a.out[(size_t)row * a.out_stride + column] = v;
}

}  // namespace

struct IrisAdapterBank {
    AdapterShape shape{};
    int16_t* weights = nullptr;
    AdapterEntry* table = nullptr;  // [slots][parts]
    uint64_t slot_weights = 0;      // weights of a slot
    uint64_t part_at[IRIS_ADAPTER_PARTS] = {};
    uint32_t most_rows = 0, width = 0;
};

extern "C" {

int iris_adapters_create(uint32_t cols, const IrisAdapterPart* parts, uint32_t part_count, uint32_t slots, uint32_t max_rank,
                         IrisAdapterBank** out) {
    if (!out) return IRIS_E_INVALID;
    *out = nullptr;
    if (!parts || !part_count || part_count > IRIS_ADAPTER_PARTS || !cols || cols % 32 || !slots || !max_rank) return IRIS_E_INVALID;
    if (cols > 65504 || slots > 65535 || max_rank > IRIS_ADAPTER_RANK) return IRIS_E_RANGE;
    for (uint32_t p = 0; p < part_count; p++) {
        if (!parts[p].rows || !parts[p].step) return IRIS_E_INVALID;
        if (parts[p].first + (uint64_t)(parts[p].rows - 1) * parts[p].step >= 1u << 24) return IRIS_E_RANGE;
    }
    // Two parts share an output where a column lies in both progressions.
    for (uint32_t p = 0; p < part_count; p++)
        for (uint32_t q = 0; q < p; q++)
            for (uint32_t i = 0; i < parts[p].rows; i++) {
                const int64_t off = (int64_t)parts[p].first + (int64_t)i * parts[p].step - parts[q].first;
                if (off >= 0 && off % parts[q].step == 0 && off / parts[q].step < parts[q].rows) return IRIS_E_INVALID;
            }
    IrisAdapterBank* b = new (std::nothrow) IrisAdapterBank();
    if (!b) return IRIS_E_NOMEM;
    AdapterShape& s = b->shape;
    s.cols = cols, s.part_count = part_count, s.slots = slots, s.max_rank = max_rank;
    for (uint32_t p = 0; p < part_count; p++) {
        s.parts[p] = parts[p];
        b->part_at[p] = b->slot_weights;
        b->slot_weights += (uint64_t)max_rank * cols + (uint64_t)parts[p].rows * stride_of(max_rank);
        b->slot_weights = (b->slot_weights + 127) & ~127ull;
        b->most_rows = std::max(b->most_rows, parts[p].rows);
        b->width = std::max(b->width, parts[p].first + (parts[p].rows - 1) * parts[p].step + 1);
    }
    const size_t entries = (size_t)slots * part_count * sizeof(AdapterEntry);
    hipError_t st = hipMalloc((void**)&b->weights, b->slot_weights * slots * 2);
    if (st == hipSuccess) st = hipMalloc((void**)&b->table, entries);
    if (st == hipSuccess) st = hipMemset(b->table, 0, entries);
    if (st == hipSuccess) st = hipDeviceSynchronize();
    if (st != hipSuccess) {
        iris_adapters_free(b);
        (void)hipGetLastError();  // returned here: not the next launch's to report
        return (int)st;
    }
    *out = b;
    return 0;
}

void iris_adapters_free(IrisAdapterBank* b) {
    if (!b) return;
    (void)hipFree(b->weights);
    (void)hipFree(b->table);
    delete b;
}

uint64_t iris_adapters_device_bytes(const IrisAdapterBank* b) {
    return b ? b->slot_weights * b->shape.slots * 2 + (uint64_t)b->shape.slots * b->shape.part_count * sizeof(AdapterEntry) : 0;
}

int iris_adapters_load(IrisAdapterBank* b, uint32_t slot, uint32_t part, const int16_t* a, uint32_t a_bits, const int16_t* w,
                       uint32_t b_bits, uint32_t rank) {
    if (!b || slot >= b->shape.slots || part >= b->shape.part_count || (rank && (!a || !w))) return IRIS_E_INVALID;
    const AdapterShape& s = b->shape;
    if (rank > s.max_rank || (rank && (a_bits > IRIS_ADAPTER_BITS || b_bits > IRIS_ADAPTER_BITS))) return IRIS_E_RANGE;
    const uint32_t rows = s.parts[part].rows, stride = stride_of(rank);
    auto past = [](const int16_t* v, uint64_t n) {
        for (uint64_t i = 0; i < n; i++)
            if (v[i] > IRIS_ADAPTER_WEIGHT || v[i] < -IRIS_ADAPTER_WEIGHT) return true;
        return false;
    };
    if (past(a, (uint64_t)rank * s.cols) || past(w, (uint64_t)rank * rows)) return IRIS_E_RANGE;
    std::vector<int16_t> padded;
    if (stride != rank) {
        try {
            padded.assign((size_t)rows * stride, 0);
        } catch (const std::bad_alloc&) {
            return IRIS_E_NOMEM;
        }
        for (uint32_t i = 0; i < rows; i++) std::memcpy(&padded[(size_t)i * stride], w + (size_t)i * rank, rank * 2);
        w = padded.data();
    }
    int16_t* to = b->weights + slot * b->slot_weights + b->part_at[part];
    AdapterEntry* entry = b->table + (size_t)slot * s.part_count + part;
    AdapterEntry e{};
    hipError_t st = hipDeviceSynchronize();
    if (st != hipSuccess) return (int)st;
    // (A copy that fails on the way leaves the part empty.)
    st = hipMemcpy(entry, &e, sizeof(e), hipMemcpyHostToDevice);
    if (st == hipSuccess && rank) {
        e.a = to, e.b = to + (((uint64_t)s.max_rank * s.cols + 7) & ~7ull);
        e.rank = rank, e.a_bits = a_bits, e.b_bits = b_bits;
        st = hipMemcpy((void*)e.a, a, (size_t)rank * s.cols * 2, hipMemcpyHostToDevice);
        if (st == hipSuccess) st = hipMemcpy((void*)e.b, w, (size_t)rows * stride * 2, hipMemcpyHostToDevice);
        if (st == hipSuccess) st = hipMemcpy(entry, &e, sizeof(e), hipMemcpyHostToDevice);
    }
    return (int)st;
}

uint64_t iris_adapters_workspace_bytes(const IrisAdapterBank* b, uint32_t rows) {
    if (!b || !rows || rows > 65535) return 0;
    return (uint64_t)rows * b->shape.part_count * b->shape.max_rank * 4;
}

int iris_adapters_apply(const IrisAdapterBank* b, const IrisAdapterRows* a, void* space, uint64_t space_bytes, void* stream) {
    if (!b || !a) return IRIS_E_INVALID;
    if (!a->rows) return 0;
    if (!a->x || !a->y || !a->out || !a->slots || !space || misaligned(a->x) || misaligned(space) || a->x_stride % 4)
        return IRIS_E_INVALID;
    const AdapterShape& s = b->shape;
    if (a->x_stride < s.cols || a->y_stride < b->width || a->out_stride < b->width) return IRIS_E_INVALID;
    if (a->out == a->y && a->out_stride != a->y_stride) return IRIS_E_INVALID;
    if (a->rows > 65535) return IRIS_E_RANGE;
    if (space_bytes < iris_adapters_workspace_bytes(b, a->rows)) return IRIS_E_RANGE;
    hipLaunchKernelGGL(shrink_row_kernel, dim3(s.part_count * s.max_rank, a->rows), dim3(256), 0, (hipStream_t)stream, *a, s,
                       b->table, (int32_t*)space);
    hipLaunchKernelGGL(expand_row_kernel, dim3((b->most_rows + 255) / 256, a->rows, s.part_count), dim3(256), 0,
                       (hipStream_t)stream, *a, s, b->table, (const int32_t*)space);
    return (int)hipGetLastError();
}

}  // extern "C"
