// The low-rank adapters of a model's layers: a bank for each product that any of
// them touches, by the DETWGT names of its parts.
#include <array>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "runtime_internal.h"

struct IrisModelAdapters {
    IrisModel* model = nullptr;
    uint32_t slots = 0, max_rank = 0;
    std::vector<std::array<IrisAdapterBank*, ADAPT_PRODUCTS>> banks;  // per layer; null: no adapter touches the product
};

namespace {

// The product that a name's suffix is a part of.
bool product_of(const char* suffix, uint32_t* product, uint32_t* part) {
    static const struct {
        const char* suffix;
        uint32_t product, part;
    } NAMES[] = {{"self_attn.q_proj.weight", ADAPT_QKV, 0}, {"self_attn.k_proj.weight", ADAPT_QKV, 1},
                 {"self_attn.v_proj.weight", ADAPT_QKV, 2}, {"self_attn.o_proj.weight", ADAPT_O, 0},
                 {"mlp.gate_proj.weight", ADAPT_GATE_UP, 0}, {"mlp.up_proj.weight", ADAPT_GATE_UP, 1},
                 {"mlp.down_proj.weight", ADAPT_DOWN, 0}};
    for (const auto& n : NAMES)
        if (!std::strcmp(n.suffix, suffix)) {
            *product = n.product, *part = n.part;
            return true;
        }
    return false;
}

}  // namespace

AdapterProductShape iris_adapter_product(const IrisModel* m, uint32_t layer, uint32_t product) {
    const LayerWeights& L = m->layers[layer];
    const uint32_t H = m->d.hidden;
    AdapterProductShape s{};
    if (product == ADAPT_QKV) {
        s.cols = H, s.part_count = 3;
        s.parts[0] = {L.q_rows, 0, 1}, s.parts[1] = {L.kv_rows, L.q_rows, 1}, s.parts[2] = {L.kv_rows, L.q_rows + L.kv_rows, 1};
    } else if (product == ADAPT_GATE_UP) {  // rows in turn, as the stacked matrix has them
        s.cols = H, s.part_count = 2;
        s.parts[0] = {L.ffn, 0, 2}, s.parts[1] = {L.ffn, 1, 2};
    } else {
        s.cols = product == ADAPT_O ? L.q_rows : L.ffn, s.part_count = 1;
        s.parts[0] = {H, 0, 1};
    }
    return s;
}

const IrisAdapterBank* iris_model_adapters_bank(const IrisModelAdapters* set, uint32_t layer, uint32_t product) {
    return set ? set->banks[layer][product] : nullptr;
}

const IrisModel* iris_model_adapters_model(const IrisModelAdapters* set, uint32_t* slots, uint32_t* max_rank) {
    *slots = set->slots, *max_rank = set->max_rank;
    return set->model;
}

extern "C" {

int iris_model_adapters_create(IrisModel* m, uint32_t slots, uint32_t max_rank, IrisModelAdapters** out) {
    if (!out) return IRIS_E_INVALID;
    *out = nullptr;
    if (!m || !m->finalized || !slots || !max_rank) return IRIS_E_INVALID;
    if (slots > 65535 || max_rank > IRIS_ADAPTER_RANK) return IRIS_E_RANGE;
    IrisModelAdapters* set = new (std::nothrow) IrisModelAdapters();
    if (!set) return IRIS_E_NOMEM;
    set->model = m, set->slots = slots, set->max_rank = max_rank;
    try {
        set->banks.assign(m->d.layers, {});
    } catch (const std::bad_alloc&) {
        delete set;
        return IRIS_E_NOMEM;
    }
    *out = set;
    return 0;
}

void iris_model_adapters_free(IrisModelAdapters* set) {
    if (!set) return;
    for (auto& layer : set->banks)
        for (IrisAdapterBank* b : layer) iris_adapters_free(b);
    delete set;
}

uint64_t iris_model_adapters_device_bytes(const IrisModelAdapters* set) {
    uint64_t bytes = 0;
    if (set)
        for (const auto& layer : set->banks)
            for (const IrisAdapterBank* b : layer) bytes += iris_adapters_device_bytes(b);
    return bytes;
}

int iris_model_adapters_load(IrisModelAdapters* set, uint32_t slot, const char* name, const int16_t* a, uint32_t a_bits,
                             const int16_t* b, uint32_t b_bits, uint32_t rank) {
    if (!set || !name || slot >= set->slots) return IRIS_E_INVALID;
    uint32_t product, part;
    int layer = -1;
    std::string suffix;
    bool whole = false;  // the name is a layer's number as it is written, and the suffix
    try {
        layer = iris_layer_of(name, &suffix);
        const std::string full = name, end = "layers." + std::to_string(layer) + "." + suffix;
        whole = layer >= 0 && full.size() >= end.size() && full.compare(full.size() - end.size(), end.size(), end) == 0;
    } catch (const std::bad_alloc&) {
        return IRIS_E_NOMEM;
    }
    if (!whole || (uint32_t)layer >= set->model->d.layers || !product_of(suffix.c_str(), &product, &part)) return IRIS_E_INVALID;
    IrisAdapterBank*& bank = set->banks[layer][product];
    if (!bank) {
        if (!rank) return 0;
        const AdapterProductShape s = iris_adapter_product(set->model, (uint32_t)layer, product);
        const int rc = iris_adapters_create(s.cols, s.parts, s.part_count, set->slots, set->max_rank, &bank);
        if (rc) return rc;
    }
    return iris_adapters_load(bank, slot, part, a, a_bits, b, b_bits, rank);
}

int iris_model_adapters_clear(IrisModelAdapters* set, uint32_t slot) {
    if (!set || slot >= set->slots) return IRIS_E_INVALID;
    for (uint32_t l = 0; l < set->banks.size(); l++)
        for (uint32_t product = 0; product < ADAPT_PRODUCTS; product++)
            if (IrisAdapterBank* bank = set->banks[l][product])
                for (uint32_t part = 0; part < iris_adapter_product(set->model, l, product).part_count; part++) {
                    const int rc = iris_adapters_load(bank, slot, part, nullptr, 0, nullptr, 0, 0);
                    if (rc) return rc;
                }
    return 0;
}

}  // extern "C"
