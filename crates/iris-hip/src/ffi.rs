//! The C ABI of libiris_hip, one declaration per function of
//! include/iris_hip.h, in the header's order. The first five are the
//! reference's own extern block (crates/inference/kernels/src/gpu.rs:45-62).

use std::os::raw::{c_char, c_int, c_void};

/// Opaque device matrix (the reference's `DeviceMatrix`, gpu.rs:40-43).
#[repr(C)]
pub struct Q8GpuMatrix {
    _private: [u8; 0],
}

#[repr(C)]
pub struct IrisModel {
    _private: [u8; 0],
}

#[repr(C)]
pub struct IrisSession {
    _private: [u8; 0],
}


#[repr(C)]
pub struct IrisBatch {
    _private: [u8; 0],
}

pub const IRIS_FAMILY_MISTRAL_DENSE: i32 = 0;
pub const IRIS_FAMILY_GEMMA_DENSE: i32 = 1;
pub const IRIS_NOALLOC_SCRATCH_BYTES: u64 = 32 << 20;

/// Shape scalars (include/iris_hip.h `IrisModelDesc`; the reference's
/// MistralShape / DirectInferShape, crates/inference/artifacts/src/direct.rs:241-290).
#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct IrisModelDesc {
    pub family: i32,
    pub hidden: u32,
    pub layers: u32,
    pub heads: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
    pub ffn: u32,
    pub vocab: u32,
    pub norm_eps: i64,
    pub attention_scale_q32: u32,
    pub max_positions: u32,
    pub tied_head: i32,
    pub global_head_dim: u32,
    pub ple_width: u32,
    pub sliding_window: u32,
    pub num_kv_shared_layers: u32,
    pub rope_base_sliding: i64,
    pub rope_base_full: i64,
    pub partial_rotary_q16: i32,
    pub embedding_scale: i32,
    pub ple_embedding_scale: i32,
    pub ple_projection_scalar: i32,
    pub ple_input_scale: i32,
    pub final_logit_softcap: i32,
    pub layer_is_sliding: *const u8,
}

/// Key and value pages of one layer (include/iris_hip.h `IrisPagedKv`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisPagedKv {
    pub k: *mut i32,
    pub v: *mut i32,
    pub pages: u32,
    pub page_size: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
}

/// The block tables and slot map of a pass (`IrisPagedPlan`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisPagedPlan {
    pub lengths: *const i32,
    pub added: *const i32,
    pub parents: *const i32,
    pub held: *const i32,
    pub held_out: *mut i32,
    pub table: *mut i32,
    pub ring: *mut i32,
    pub ring_state: *const i32,
    pub ring_state_out: *mut i32,
    pub row_start: *mut i32,
    pub slots: *mut i32,
    pub positions: *mut i32,
    pub status: *mut i32,
    pub requests: u32,
    pub table_stride: u32,
    pub pages: u32,
    pub page_size: u32,
    pub max_rows: u32,
}

/// Causal attention over packed prompts (`IrisPackedAttention`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisPackedAttention {
    pub q: *const i32,
    pub k: *const i32,
    pub v: *const i32,
    pub out: *mut i32,
    pub row_start: *const i32,
    pub status: *mut i32,
    pub q_stride: u32,
    pub k_stride: u32,
    pub v_stride: u32,
    pub out_stride: u32,
    pub sequences: u32,
    pub rows: u32,
    pub max_length: u32,
    pub heads: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
    pub window: u32,
    pub scaled: i32,
    pub scale_q32: u32,
}

/// Attention of drafted trees over the paged cache (`IrisTreeAttention`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisTreeAttention {
    pub q: *const i32,
    pub out: *mut i32,
    pub row_start: *const i32,
    pub lengths: *const i32,
    pub parents: *const i32,
    pub table: *const i32,
    pub status: *mut i32,
    pub q_stride: u32,
    pub out_stride: u32,
    pub requests: u32,
    pub rows: u32,
    pub table_stride: u32,
    pub max_nodes: u32,
    pub max_positions: u32,
    pub heads: u32,
    pub window: u32,
    pub scaled: i32,
    pub scale_q32: u32,
}

/// The header's 16-bit integers, by its own name for them.
#[allow(non_camel_case_types)]
pub type int16_t = i16;

/// A product's part for its adapters: output i is column first + i * step
/// (include/iris_hip.h `IrisAdapterPart`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisAdapterPart {
    pub rows: u32,
    pub first: u32,
    pub step: u32,
}

/// The low-rank adapters of one product on the device.
#[repr(C)]
pub struct IrisAdapterBank {
    _private: [u8; 0],
}

/// The low-rank adapters of a model's layers.
#[repr(C)]
pub struct IrisModelAdapters {
    _private: [u8; 0],
}

/// Rows with an adapter each (`IrisAdapterRows`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisAdapterRows {
    pub x: *const i32,
    pub y: *const i32,
    pub out: *mut i32,
    pub slots: *const i32,
    pub status: *mut i32,
    pub x_stride: u32,
    pub y_stride: u32,
    pub out_stride: u32,
    pub rows: u32,
}

/// One request's penalties and biases (`IrisTokenRule`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisTokenRule {
    pub repetition: i32,
    pub frequency: i32,
    pub presence: i32,
    pub window: u32,
    pub bias_start: u32,
    pub bias_count: u32,
}

/// Rules on rows of logits (`IrisLogitsRules`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisLogitsRules {
    pub logits: *const i32,
    pub out: *mut i32,
    pub request: *const i32,
    pub rules: *const IrisTokenRule,
    pub history: *const i32,
    pub lengths: *const i32,
    pub row_start: *const i32,
    pub ids: *const i32,
    pub parents: *const i32,
    pub bias_ids: *const i32,
    pub bias_values: *const i32,
    pub masks: *const u32,
    pub mask_of: *const i32,
    pub status: *mut i32,
    pub rows: u32,
    pub first_row: u32,
    pub vocab: u32,
    pub logits_stride: u32,
    pub out_stride: u32,
    pub requests: u32,
    pub history_stride: u32,
    pub biases: u32,
    pub mask_rows: u32,
    pub mask_stride: u32,
}

/// How a request draws its tokens (`IrisDrawing`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisDrawing {
    pub inverse_temperature: i32,
    pub top_k: u32,
    pub top_p: u32,
    pub max_gap: u32,
}

/// A token for each row of logits (`IrisLogitsDraw`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct IrisLogitsDraw {
    pub logits: *const i32,
    pub request: *const i32,
    pub drawings: *const IrisDrawing,
    pub numbers: *const u32,
    pub tokens: *mut i32,
    pub mass: *mut i64,
    pub status: *mut i32,
    pub rows: u32,
    pub vocab: u32,
    pub logits_stride: u32,
    pub requests: u32,
}

extern "C" {
    pub fn q8gpu_error(code: c_int) -> *const c_char;
    pub fn q8gpu_init() -> c_int;
    pub fn q8gpu_upload(
        weights: *const i8,
        scales: *const i64,
        rows: u32,
        cols: u32,
        out: *mut *mut Q8GpuMatrix,
    ) -> c_int;
    pub fn q8gpu_free(matrix: *mut Q8GpuMatrix);
    pub fn q8gpu_product(matrix: *const Q8GpuMatrix, activations: *const i32, tokens: u32, out: *mut i32) -> c_int;

    pub fn q8gpu_upload_q8_0(blocks: *const u8, rows: u32, cols: u32, out: *mut *mut Q8GpuMatrix) -> c_int;
    pub fn q8gpu_product_device(
        matrix: *const Q8GpuMatrix,
        d_activations: *const i32,
        tokens: u32,
        d_out: *mut i32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn q8gpu_workspace_bytes(matrix: *const Q8GpuMatrix, tokens: u32) -> u64;
    pub fn q8gpu_product_device_ws(
        matrix: *const Q8GpuMatrix,
        d_activations: *const i32,
        tokens: u32,
        d_out: *mut i32,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn q8gpu_prepare_matrix_cores(matrix: *mut Q8GpuMatrix, stream: *mut c_void) -> c_int;
    pub fn q8gpu_product_device_noalloc(
        matrix: *const Q8GpuMatrix,
        d_activations: *const i32,
        tokens: u32,
        d_out: *mut i32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn q8gpu_matrix_info(
        matrix: *const Q8GpuMatrix,
        rows: *mut u32,
        cols: *mut u32,
        scale_mode: *mut c_int,
        bytes: *mut u64,
    ) -> c_int;
    pub fn iris_product_route(matrix: *const Q8GpuMatrix, tokens: u32, name: *mut c_char, size: u32) -> c_int;
    pub fn q8gpu_synchronize() -> c_int;

    pub fn iris_device_malloc(bytes: u64, out: *mut *mut c_void) -> c_int;
    pub fn iris_device_free(ptr: *mut c_void) -> c_int;
    pub fn iris_memcpy_h2d(dst: *mut c_void, src: *const c_void, bytes: u64) -> c_int;
    pub fn iris_memcpy_d2h(dst: *mut c_void, src: *const c_void, bytes: u64) -> c_int;
    pub fn iris_memcpy_d2d(dst: *mut c_void, src: *const c_void, bytes: u64) -> c_int;
    pub fn iris_probe_hbm_read(d_buf: *const c_void, bytes: u64, repeats: u32, gb_per_s: *mut f64) -> c_int;
    pub fn iris_probe_mfma_i8(random_operands: u32, iterations: u32, tops: *mut f64) -> c_int;
    pub fn iris_probe_handoff(workgroups: u32, round_trip_us: *mut f64, atomic_us: *mut f64, barrier_us: *mut f64)
        -> c_int;
    pub fn iris_probe_row_latency(flood_waves: u32, vector_us: *mut f64, scalar_us: *mut f64) -> c_int;
    pub fn iris_time_product(
        matrices: *const *const Q8GpuMatrix,
        count: u32,
        d_activations: *const i32,
        tokens: u32,
        d_out: *mut i32,
        iterations: u32,
        ms_per_product: *mut f64,
    ) -> c_int;
    pub fn iris_time_bcast_product(
        matrices: *const *const Q8GpuMatrix,
        count: u32,
        d_activations: *const i32,
        d_out: *mut i32,
        iterations: u32,
        ms_per_product: *mut f64,
    ) -> c_int;
    pub fn iris_time_product_ws(
        matrix: *const Q8GpuMatrix,
        d_activations: *const i32,
        tokens: u32,
        d_out: *mut i32,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        iterations: u32,
        ms_per_product: *mut f64,
    ) -> c_int;

    pub fn iris_model_create(desc: *const IrisModelDesc, out: *mut *mut IrisModel) -> c_int;
    pub fn iris_model_set_tensor(
        model: *mut IrisModel,
        name: *const c_char,
        width: i32,
        data: *const c_void,
        rows: u64,
        cols: u64,
    ) -> c_int;
    pub fn iris_model_finalize(model: *mut IrisModel) -> c_int;
    pub fn iris_model_free(model: *mut IrisModel);
    pub fn iris_model_device_bytes(model: *const IrisModel) -> u64;
    pub fn iris_model_ids_refused(model: *const IrisModel, ids: *const i32, count: u32, at: *mut u32) -> c_int;

    pub fn iris_session_create(
        model: *mut IrisModel,
        max_positions: u32,
        max_rows: u32,
        out: *mut *mut IrisSession,
    ) -> c_int;
    pub fn iris_session_free(session: *mut IrisSession);
    pub fn iris_session_generate(
        session: *mut IrisSession,
        prompt: *const i32,
        prompt_len: u32,
        tokens: u32,
        eos_ids: *const i32,
        n_eos: u32,
        out_tokens: *mut i32,
        out_count: *mut u32,
        out_logits: *mut i32,
        use_graph: i32,
    ) -> c_int;
    pub fn iris_session_layer_pass(
        session: *mut IrisSession,
        ids: *const i32,
        count: u32,
        out_rows: *mut i32,
        out_hashes: *mut u8,
    ) -> c_int;
    pub fn iris_session_layer_range(
        session: *mut IrisSession,
        ids: *const i32,
        count: u32,
        start_position: u32,
        out_rows: *mut i32,
        out_hashes: *mut u8,
    ) -> c_int;
    pub fn iris_session_layer_stage(
        session: *mut IrisSession,
        layer: u32,
        in_rows: *const i32,
        count: u32,
        start_position: u32,
        ple_rows: *const i32,
        out_rows: *mut i32,
    ) -> c_int;
    pub fn iris_session_write_kv(
        session: *mut IrisSession,
        layer: u32,
        pos0: u32,
        count: u32,
        k: *const i32,
        v: *const i32,
    ) -> c_int;
    pub fn iris_session_read_kv(
        session: *mut IrisSession,
        layer: u32,
        pos0: u32,
        count: u32,
        k_out: *mut i32,
        v_out: *mut i32,
    ) -> c_int;
    pub fn iris_session_time_decode(
        session: *mut IrisSession,
        prompt: *const i32,
        prompt_len: u32,
        steps: u32,
        ms_per_token: *mut f64,
        prefill_ms: *mut f64,
        out_tokens: *mut i32,
    ) -> c_int;
    pub fn iris_session_time_decode_launches(
        session: *mut IrisSession,
        prompt: *const i32,
        prompt_len: u32,
        steps: u32,
        use_graph: c_int,
        ms_per_token: *mut f64,
        prefill_ms: *mut f64,
        out_tokens: *mut i32,
    ) -> c_int;
    pub fn iris_kernel_tracer_loaded() -> c_int;
    pub fn iris_session_time_pass(session: *mut IrisSession, ids: *const i32, count: u32, ms: *mut f64) -> c_int;
    pub fn iris_attention_numerics(
        diff: *const u32,
        e: *const u64,
        sum: *const u64,
        dot: *const i64,
        scale_q32: u32,
        n: u32,
        exp_out: *mut u64,
        weight_out: *mut i32,
        score_out: *mut i32,
    ) -> c_int;
    pub fn iris_score_numerics(
        dot: *const i64,
        scaled: c_int,
        scale_q32: u32,
        n: u32,
        score_out: *mut i32,
        quick_out: *mut i32,
    ) -> c_int;
    pub fn iris_silu_device(x: *const i32, n: u32, out: *mut i32) -> c_int;
    pub fn iris_silu_table_device(x: *const i32, n: u32, out: *mut i32) -> c_int;
    pub fn iris_paged_plan(plan: *const IrisPagedPlan, stream: *mut c_void) -> c_int;
    pub fn iris_paged_store(
        cache: *const IrisPagedKv,
        k: *const i32,
        k_stride: u32,
        v: *const i32,
        v_stride: u32,
        slots: *const i32,
        rows: u32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn iris_attention_packed_workspace_bytes(a: *const IrisPackedAttention) -> u64;
    pub fn iris_attention_packed(
        a: *const IrisPackedAttention,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn iris_attention_tree_workspace_bytes(cache: *const IrisPagedKv, a: *const IrisTreeAttention) -> u64;
    pub fn iris_attention_tree(
        cache: *const IrisPagedKv,
        a: *const IrisTreeAttention,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn iris_adapters_create(
        cols: u32,
        parts: *const IrisAdapterPart,
        part_count: u32,
        slots: u32,
        max_rank: u32,
        out: *mut *mut IrisAdapterBank,
    ) -> c_int;
    pub fn iris_adapters_free(bank: *mut IrisAdapterBank);
    pub fn iris_adapters_device_bytes(bank: *const IrisAdapterBank) -> u64;
    pub fn iris_adapters_load(
        bank: *mut IrisAdapterBank,
        slot: u32,
        part: u32,
        a: *const int16_t,
        a_bits: u32,
        b: *const int16_t,
        b_bits: u32,
        rank: u32,
    ) -> c_int;
    pub fn iris_adapters_workspace_bytes(bank: *const IrisAdapterBank, rows: u32) -> u64;
    pub fn iris_adapters_apply(
        bank: *const IrisAdapterBank,
        a: *const IrisAdapterRows,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn iris_logits_rules(a: *const IrisLogitsRules, stream: *mut c_void) -> c_int;
    pub fn iris_logits_draw_workspace_bytes(a: *const IrisLogitsDraw) -> u64;
    pub fn iris_logits_draw(
        a: *const IrisLogitsDraw,
        d_workspace: *mut c_void,
        workspace_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn iris_batch_create(
        model: *mut IrisModel,
        requests: u32,
        pages: u32,
        page_size: u32,
        max_positions: u32,
        max_rows: u32,
        out: *mut *mut IrisBatch,
    ) -> c_int;
    pub fn iris_batch_free(batch: *mut IrisBatch);
    pub fn iris_batch_prefill(
        batch: *mut IrisBatch,
        ids: *const i32,
        counts: *const u32,
        out_tokens: *mut i32,
    ) -> c_int;
    pub fn iris_batch_step(
        batch: *mut IrisBatch,
        ids: *const i32,
        parents: *const i32,
        counts: *const u32,
        out_tokens: *mut i32,
        out_kept: *mut u32,
    ) -> c_int;
    pub fn iris_batch_release(batch: *mut IrisBatch, request: u32) -> c_int;
    pub fn iris_batch_length(batch: *const IrisBatch, request: u32, out: *mut u32) -> c_int;
    pub fn iris_model_adapters_create(
        model: *mut IrisModel,
        slots: u32,
        max_rank: u32,
        out: *mut *mut IrisModelAdapters,
    ) -> c_int;
    pub fn iris_model_adapters_free(set: *mut IrisModelAdapters);
    pub fn iris_model_adapters_device_bytes(set: *const IrisModelAdapters) -> u64;
    pub fn iris_model_adapters_load(
        set: *mut IrisModelAdapters,
        slot: u32,
        name: *const c_char,
        a: *const int16_t,
        a_bits: u32,
        b: *const int16_t,
        b_bits: u32,
        rank: u32,
    ) -> c_int;
    pub fn iris_model_adapters_clear(set: *mut IrisModelAdapters, slot: u32) -> c_int;
    pub fn iris_batch_adapters(batch: *mut IrisBatch, set: *const IrisModelAdapters) -> c_int;
    pub fn iris_batch_adapter(batch: *mut IrisBatch, request: u32, slot: i32) -> c_int;
    pub fn iris_batch_rule(
        batch: *mut IrisBatch,
        request: u32,
        rule: *const IrisTokenRule,
        bias_ids: *const i32,
        bias_values: *const i32,
    ) -> c_int;
    pub fn iris_batch_drawing(
        batch: *mut IrisBatch,
        request: u32,
        drawing: *const IrisDrawing,
        numbers: *const u32,
        first: u32,
        count: u32,
    ) -> c_int;
    pub fn iris_batch_masks(
        batch: *mut IrisBatch,
        masks: *const u32,
        mask_rows: u32,
        mask_of: *const i32,
        rows: u32,
    ) -> c_int;
    pub fn iris_sha256_bytes(data: *const u8, len: u64, out: *mut u8) -> c_int;
}
