// Generated by gen_ffi.py from include/hipml_cuda.h: do not edit by hand.
// Raw bindings of libhipml_cuda.so, the counterpart of crates/hipml-hip/src/ffi.rs:29-105
// plus the attention launchers (section B of the header).
#![allow(non_camel_case_types)]
use std::ffi::{c_char, c_int, c_uint, c_void};

pub type Status = c_int; // 0 = success
pub type Stream = *mut c_void;
pub type Event = *mut c_void;
pub type Graph = *mut c_void;
pub type GraphExec = *mut c_void;
pub type Module = *mut c_void;
pub type Function = *mut c_void;

#[link(name = "hipml_cuda")]
extern "C" {
    pub fn hipml_init(flags: c_uint) -> Status;
    pub fn hipml_get_device_count(count: *mut c_int) -> Status;
    pub fn hipml_get_device(device: *mut c_int, ordinal: c_int) -> Status;
    pub fn hipml_set_device(device: c_int) -> Status;
    pub fn hipml_device_get_name(name: *mut c_char, len: c_int, device: c_int) -> Status;
    pub fn hipml_device_total_mem(bytes: *mut usize, device: c_int) -> Status;
    pub fn hipml_device_compute_capability(major: *mut c_int, minor: *mut c_int, device: c_int) -> Status;
    pub fn hipml_get_error_string(code: c_int) -> *const c_char;
    pub fn hipml_last_error_message() -> *const c_char;
    pub fn hipml_malloc(ptr: *mut *mut c_void, size: usize) -> Status;
    pub fn hipml_free(ptr: *mut c_void) -> Status;
    pub fn hipml_memset(dst: *mut c_void, value: c_int, size: usize) -> Status;
    pub fn hipml_mem_get_info(free_bytes: *mut usize, total_bytes: *mut usize) -> Status;
    pub fn hipml_memcpy(dst: *mut c_void, src: *const c_void, size: usize, kind: c_int) -> Status;
    pub fn hipml_memcpy_async(dst: *mut c_void, src: *const c_void, size: usize, kind: c_int, stream: Stream) -> Status;
    pub fn hipml_device_synchronize() -> Status;
    pub fn hipml_host_alloc(ptr: *mut *mut c_void, size: usize) -> Status;
    pub fn hipml_host_free(ptr: *mut c_void) -> Status;
    pub fn hipml_event_create(event: *mut Event) -> Status;
    pub fn hipml_event_destroy(event: Event) -> Status;
    pub fn hipml_event_record(event: Event, stream: Stream) -> Status;
    pub fn hipml_event_synchronize(event: Event) -> Status;
    pub fn hipml_event_elapsed_time(ms: *mut f32, start: Event, stop: Event) -> Status;
    pub fn hipml_stream_create(stream: *mut Stream) -> Status;
    pub fn hipml_stream_destroy(stream: Stream) -> Status;
    pub fn hipml_stream_synchronize(stream: Stream) -> Status;
    pub fn hipml_stream_wait_event(stream: Stream, event: Event, flags: c_uint) -> Status;
    pub fn hipml_stream_begin_capture(stream: Stream, mode: c_int) -> Status;
    pub fn hipml_stream_end_capture(stream: Stream, graph: *mut Graph) -> Status;
    pub fn hipml_graph_instantiate(exec: *mut GraphExec, graph: Graph, error_node: *mut c_void, log_buffer: *mut c_char, log_size: usize) -> Status;
    pub fn hipml_graph_launch(exec: GraphExec, stream: Stream) -> Status;
    pub fn hipml_graph_upload(exec: GraphExec, stream: Stream) -> Status;
    pub fn hipml_graph_destroy(graph: Graph) -> Status;
    pub fn hipml_graph_exec_destroy(exec: GraphExec) -> Status;
    pub fn hipml_module_load(module: *mut Module, file: *const c_char) -> Status;
    pub fn hipml_module_unload(module: Module) -> Status;
    pub fn hipml_module_get_function(function: *mut Function, module: Module, name: *const c_char) -> Status;
    pub fn hipml_module_launch_kernel(function: Function, grid_x: c_uint, grid_y: c_uint, grid_z: c_uint, block_x: c_uint, block_y: c_uint, block_z: c_uint, shared_mem_bytes: c_uint, stream: Stream, kernel_params: *mut *mut c_void, extra: *mut *mut c_void) -> Status;
    pub fn hipml_kv_encode(stream: Stream, step: *const c_int, dtype: c_int, k_row: *const f32, v_row: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, n_kv: c_int, head_dim: c_int, stride: c_int) -> Status;
    pub fn hipml_kv_encode_bulk(stream: Stream, dtype: c_int, k_f32: *const f32, v_f32: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, n_kv: c_int, head_dim: c_int, stride: c_int, start: c_int, src0: c_int, rows: c_int) -> Status;
    pub fn hipml_kv_encode_rows(stream: Stream, dtype: c_int, k_f32: *const f32, v_f32: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, n_kv: c_int, head_dim: c_int, stride: c_int, pos: *const c_int, slot_bytes: c_int, slots: c_int) -> Status;
    pub fn hipml_kv_append_f32(stream: Stream, step: *const c_int, k_cache: *mut f32, v_cache: *mut f32, k_row: *const f32, v_row: *const f32, width: c_int) -> Status;
    pub fn hipml_kv_append_chunk_f32(stream: Stream, k_cache: *mut f32, v_cache: *mut f32, k: *const f32, v: *const f32, pos0: c_int, width: c_int, tokens: c_int) -> Status;
    pub fn hipml_attn_decode_kv(stream: Stream, step: *const c_int, selector: c_int, q: *const f32, k: *const c_void, v: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize) -> Status;
    pub fn hipml_attn_decode_cols_f32(stream: Stream, q: *const f32, k_cache: *const f32, v_cache: *const f32, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, n_ctx: c_int, pos0: c_int, rows: c_int) -> Status;
    pub fn hipml_kv_append_cols_f32(stream: Stream, k_cache: *mut f32, v_cache: *mut f32, k: *const f32, v: *const f32, pos0: c_int, rows: c_int, width: c_int) -> Status;
    pub fn hipml_attn_decode_cols(stream: Stream, selector: c_int, pos: *const c_int, q: *const f32, k: *const c_void, v: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, cols: c_int, acc_slot: c_int, ml_slot: c_int, q_slot: c_int) -> Status;
    pub fn hipml_kv_rows_copy(stream: Stream, dst: *mut c_void, src: *const c_void, n_kv: c_int, row_bytes: c_int, dst_stride: c_int, src_stride: c_int, rows: c_int) -> Status;
    pub fn hipml_attn_decode_kv_gated(stream: Stream, step: *const c_int, selector: c_int, q: *const f32, k: *const c_void, v: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, gate: *const f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize) -> Status;
    pub fn hipml_attn_decode_kv_append(stream: Stream, step: *const c_int, selector: c_int, k_row: *const f32, v_row: *const f32, q: *const f32, k: *mut c_void, v: *mut c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, gate: *const f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize) -> Status;
    pub fn hipml_attn_decode_batch_append(stream: Stream, dtype: c_int, pos: *const c_int, k_f32: *const f32, v_f32: *const f32, q: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, kv_slot_bytes: c_int, acc_slot: c_int, ml_slot: c_int, q_slot: c_int, slots: c_int) -> Status;
    pub fn hipml_attn_front(stream: Stream, qg: *const f32, q: *mut f32, gate: *mut f32, k: *mut f32, q_norm: *const f32, k_norm: *const f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, n_rot: c_int, sections: *const c_int, pos: *const c_int, theta_base: f32, eps: f32) -> Status;
    pub fn hipml_qg_split_chunk(stream: Stream, qg: *const f32, q: *mut f32, gate: *mut f32, n_heads: c_int, head_dim: c_int, tokens: c_int) -> Status;
    pub fn hipml_norm_rope_chunk(stream: Stream, q: *mut f32, k: *mut f32, q_norm: *const f32, k_norm: *const f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, n_rot: c_int, theta_base: f32, eps: f32, pos0: c_int, tokens: c_int) -> Status;
    pub fn hipml_q_gate(stream: Stream, q: *const f32, gate: *const f32, y: *mut f32, n: i64) -> Status;
    pub fn hipml_attn_front_append_q8(stream: Stream, qg: *const f32, k: *const f32, v: *const f32, q: *mut f32, gate: *mut f32, k_out: *mut f32, q_norm: *const f32, k_norm: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, n_heads: c_int, n_kv: c_int, head_dim: c_int, n_rot: c_int, sections: *const c_int, pos: *const c_int, step: *const c_int, pos0: c_int, tokens: c_int, stride: c_int, theta_base: f32, eps: f32) -> Status;
    pub fn hipml_attn_decode_kv_shard(stream: Stream, step: *const c_int, selector: c_int, q: *const f32, k: *const c_void, v: *const c_void, part_acc: *mut f32, part_ml: *mut f32, shard_out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize) -> Status;
    pub fn hipml_attn_decode_combine(stream: Stream, gathered: *const f32, out: *mut f32, n_heads: c_int, head_dim: c_int, shards: c_int) -> Status;
    pub fn hipml_decode_exchange_bytes(n_heads: c_int, head_dim: c_int, shards: c_int) -> usize;
    pub fn hipml_attn_decode_kv_shard_exchange(stream: Stream, step: *const c_int, selector: c_int, q: *const f32, k: *const c_void, v: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize, peer_ws: *const *mut c_void, shards: c_int, rank: c_int, phases: c_int, wait_limit_us: c_uint) -> Status;
    pub fn hipml_attn_decode_kv_shard_exchange_append(stream: Stream, step: *const c_int, selector: c_int, k_row: *const f32, v_row: *const f32, q: *const f32, k: *mut c_void, v: *mut c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize, peer_ws: *const *mut c_void, shards: c_int, rank: c_int, phases: c_int, wait_limit_us: c_uint) -> Status;
    pub fn hipml_attn_decode_kv_static(stream: Stream, step: *const c_int, selector: c_int, q: *const f32, k: *const c_void, v: *const c_void, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, k_off: usize, v_off: usize) -> Status;
    pub fn hipml_attn_decode_rows(stream: Stream, dtype: c_int, pos: *const c_int, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, kv_slot_bytes: c_int, acc_slot: c_int, ml_slot: c_int, q_slot: c_int, slots: c_int) -> Status;
    pub fn hipml_attn_decode_batch(stream: Stream, dtype: c_int, pos: *const c_int, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, part_acc: *mut f32, part_ml: *mut f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, splits: c_int, kv_slot_bytes: c_int, acc_slot: c_int, ml_slot: c_int, q_slot: c_int, slots: c_int, live_seq: c_int) -> Status;
    pub fn hipml_attn_chunk_workspace_bytes(n_kv: c_int, head_dim: c_int, pos0: c_int, tokens: c_int) -> usize;
    pub fn hipml_attn_chunk(stream: Stream, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, pos0: c_int, tokens: c_int, kv_dtype: c_int, stride: c_int, part_acc: *mut f32, part_ml: *mut f32, splits: c_int, mode: c_int, workspace: *mut c_void, workspace_bytes: usize) -> Status;
    pub fn hipml_attn_chunk_stage(stream: Stream, k_cache: *const c_void, v_cache: *const c_void, n_kv: c_int, head_dim: c_int, kv_dtype: c_int, stride: c_int, key_from: c_int, key_to: c_int, key_capacity: c_int, workspace: *mut c_void, workspace_bytes: usize) -> Status;
    pub fn hipml_attn_chunk_staged(stream: Stream, q: *const f32, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, pos0: c_int, tokens: c_int, part_acc: *mut f32, part_ml: *mut f32, splits: c_int, mode: c_int, key_capacity: c_int, workspace: *mut c_void, workspace_bytes: usize) -> Status;
    pub fn hipml_attn_chunk_staged_gated(stream: Stream, q: *const f32, out: *mut f32, gate: *const f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, pos0: c_int, tokens: c_int, part_acc: *mut f32, part_ml: *mut f32, splits: c_int, mode: c_int, key_capacity: c_int, workspace: *mut c_void, workspace_bytes: usize) -> Status;
    pub fn hipml_attn_tree_workspace_bytes(n_heads: c_int, n_kv: c_int, head_dim: c_int, nodes: c_int, slots: c_int) -> usize;
    pub fn hipml_attn_tree(stream: Stream, kv_dtype: c_int, pos: *const c_int, parents: *const c_int, q: *const f32, k_cache: *const c_void, v_cache: *const c_void, out: *mut f32, n_heads: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, scale: f32, nodes: c_int, slots: c_int, kv_slot_bytes: usize, workspace: *mut c_void, workspace_bytes: usize) -> Status;
    pub fn hipml_tree_verify(stream: Stream, pos: *const c_int, parents: *const c_int, tokens: *const c_int, target: *const f32, draft: *const f32, uniform: *const f32, path: *mut c_int, count: *mut c_int, next: *mut c_int, nodes: c_int, slots: c_int, vocab: c_int, row_stride: i64) -> Status;
    pub fn hipml_tree_verify_within(stream: Stream, pos: *const c_int, parents: *const c_int, tokens: *const c_int, target: *const f32, draft: *const f32, uniform: *const f32, path: *mut c_int, count: *mut c_int, next: *mut c_int, nodes: c_int, slots: c_int, vocab: c_int, row_stride: i64, stride: c_int) -> Status;
    pub fn hipml_kv_path_keep(stream: Stream, kv_dtype: c_int, pos: *const c_int, path: *const c_int, count: *const c_int, k_caches: *const *mut c_void, v_caches: *const *mut c_void, layers: c_int, n_kv: c_int, head_dim: c_int, stride: c_int, nodes: c_int, slots: c_int, kv_slot_bytes: usize) -> Status;
    pub fn hipml_set_decode_cta_slots(slots: c_int) -> Status;
    pub fn hipml_set_decode_body(body: c_int) -> Status;
    pub fn hipml_set_decode_fold_mode(mode: c_int) -> Status;
    pub fn hipml_decode_plan_quota(lens: *const c_int, slots: c_int, splits: c_int, n_kv: c_int, cta_slots: c_int) -> Status;
    pub fn hipml_check_device_status(stream: Stream, status: *mut c_int) -> Status;
    pub fn hipml_version() -> *const c_char;
}
