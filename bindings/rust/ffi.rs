// GENERATED by tools/gen_rust_ffi.py from include/arrow_gpu.h — do not edit; re-run the script when the header changes.
// `extern "C"` image of libarrow_gpu_hip.so's C ABI: what crates/array/src/gpu_utils/ binds instead of wgpu
// [replaces the wgpu Device / Queue / CommandEncoder calls of gpu_device.rs:29-514 and compute_pipeline.rs:8-300].
// NOT COMPILED in the build image (no rustc); tests/test_capi_symbols.py checks it against the header mechanically.
#![allow(non_camel_case_types, non_upper_case_globals, dead_code)]
use std::os::raw::{c_char, c_int, c_void};

pub const AGPU_ABI_VERSION: i32 = 2;
pub const AGPU_MAILBOX_MAX_BYTES: usize = 3840;
pub const AGPU_CHAIN_MAX_STEPS: usize = 8;
pub const AGPU_CAST_CHAIN_MAX_ARRAYS: i32 = 4;
pub const AGPU_COMM_ID_BYTES: usize = 128;
pub const ARROW_FLAG_DICTIONARY_ORDERED: i64 = 1;
pub const ARROW_FLAG_NULLABLE: i64 = 2;
pub const ARROW_FLAG_MAP_KEYS_SORTED: i64 = 4;

pub type agpu_status = i32;
pub const AGPU_OK: agpu_status = 0;
pub const AGPU_ERR_UNSUPPORTED: agpu_status = 1;
pub const AGPU_ERR_SHAPE: agpu_status = 2;
pub const AGPU_ERR_HIP: agpu_status = 3;
pub const AGPU_ERR_ARG: agpu_status = 4;
pub const AGPU_ERR_NO_DEVICE: agpu_status = 5;
pub type agpu_dtype = i32;
pub const AGPU_BOOL: agpu_dtype = 0;
pub const AGPU_F32: agpu_dtype = 1;
pub const AGPU_U32: agpu_dtype = 2;
pub const AGPU_U16: agpu_dtype = 3;
pub const AGPU_U8: agpu_dtype = 4;
pub const AGPU_I32: agpu_dtype = 5;
pub const AGPU_I16: agpu_dtype = 6;
pub const AGPU_I8: agpu_dtype = 7;
pub const AGPU_DATE32: agpu_dtype = 8;
pub type agpu_binary_op = i32;
pub const AGPU_OP_ADD: agpu_binary_op = 0;
pub const AGPU_OP_SUB: agpu_binary_op = 1;
pub const AGPU_OP_MUL: agpu_binary_op = 2;
pub const AGPU_OP_DIV: agpu_binary_op = 3;
pub const AGPU_OP_REM: agpu_binary_op = 4;
pub const AGPU_OP_MIN: agpu_binary_op = 5;
pub const AGPU_OP_MAX: agpu_binary_op = 6;
pub const AGPU_OP_AND: agpu_binary_op = 7;
pub const AGPU_OP_OR: agpu_binary_op = 8;
pub const AGPU_OP_XOR: agpu_binary_op = 9;
pub const AGPU_OP_SHL: agpu_binary_op = 10;
pub const AGPU_OP_SHR: agpu_binary_op = 11;
pub const AGPU_OP_POW: agpu_binary_op = 12;
pub type agpu_unary_op = i32;
pub const AGPU_UN_NEG: agpu_unary_op = 0;
pub const AGPU_UN_ABS: agpu_unary_op = 1;
pub const AGPU_UN_NOT: agpu_unary_op = 2;
pub const AGPU_UN_SQRT: agpu_unary_op = 3;
pub const AGPU_UN_CBRT: agpu_unary_op = 4;
pub const AGPU_UN_EXP: agpu_unary_op = 5;
pub const AGPU_UN_EXP2: agpu_unary_op = 6;
pub const AGPU_UN_LOG: agpu_unary_op = 7;
pub const AGPU_UN_LOG2: agpu_unary_op = 8;
pub const AGPU_UN_SIN: agpu_unary_op = 9;
pub const AGPU_UN_COS: agpu_unary_op = 10;
pub const AGPU_UN_ACOS: agpu_unary_op = 11;
pub const AGPU_UN_SINH: agpu_unary_op = 12;
pub const AGPU_UN_POPCOUNT: agpu_unary_op = 13;
pub type agpu_cmp_op = i32;
pub const AGPU_CMP_GT: agpu_cmp_op = 0;
pub const AGPU_CMP_GTEQ: agpu_cmp_op = 1;
pub const AGPU_CMP_LT: agpu_cmp_op = 2;
pub const AGPU_CMP_LTEQ: agpu_cmp_op = 3;
pub const AGPU_CMP_EQ: agpu_cmp_op = 4;
pub type agpu_reduce_op = i32;
pub const AGPU_RED_SUM: agpu_reduce_op = 0;
pub const AGPU_RED_MIN: agpu_reduce_op = 1;
pub const AGPU_RED_MAX: agpu_reduce_op = 2;
pub type agpu_chain_kind = i32;
pub const AGPU_CHAIN_UNARY: agpu_chain_kind = 0;
pub const AGPU_CHAIN_SCALAR: agpu_chain_kind = 1;
pub const AGPU_CHAIN_ARRAY: agpu_chain_kind = 2;
pub type agpu_row_type = i32;
pub const AGPU_ROW_F32: agpu_row_type = 0;
pub const AGPU_ROW_F16: agpu_row_type = 1;
pub const AGPU_ROW_BF16: agpu_row_type = 2;
pub type agpu_code_type = i32;
pub const AGPU_CODE_I8: agpu_code_type = 0;
pub const AGPU_CODE_I4: agpu_code_type = 1;
pub const AGPU_CODE_E4M3: agpu_code_type = 2;
pub type agpu_comm_dtype = i32;
pub const AGPU_COMM_F32: agpu_comm_dtype = 0;
pub const AGPU_COMM_F64: agpu_comm_dtype = 1;
pub const AGPU_COMM_I32: agpu_comm_dtype = 2;
pub const AGPU_COMM_U32: agpu_comm_dtype = 3;
pub const AGPU_COMM_I64: agpu_comm_dtype = 4;
pub const AGPU_COMM_U64: agpu_comm_dtype = 5;

#[repr(C)] pub struct agpu_device { _private: [u8; 0] }
#[repr(C)] pub struct agpu_pipeline { _private: [u8; 0] }
#[repr(C)] pub struct agpu_event { _private: [u8; 0] }
#[repr(C)] pub struct agpu_graph { _private: [u8; 0] }
#[repr(C)] pub struct agpu_comm { _private: [u8; 0] }
#[repr(C)] pub struct agpu_ipc_reader { _private: [u8; 0] }
#[repr(C)] pub struct agpu_ipc_writer { _private: [u8; 0] }

#[repr(C)]
pub struct agpu_chain_step {
    pub op: i32,
    pub kind: i32,
    pub operand: *const c_void,
}
#[repr(C)]
pub struct agpu_f32_stats {
    pub sum: f32,
    pub min: f32,
    pub max: f32,
    pub reserved: u32,
    pub sum_f64: f64,
}
#[repr(C)]
pub struct agpu_rows {
    pub data: *mut c_void,
    pub row_stride: u64,
    pub head_stride: u64,
    pub row_type: i32,
}
#[repr(C)]
pub struct agpu_quantised_rows {
    pub codes: *mut c_void,
    pub scales: *mut f32,
    pub n_slots: u64,
    pub heads: u32,
    pub dim: u32,
    pub group: u32,
    pub code: i32,
}
#[repr(C)]
pub struct agpu_page_map {
    pub tables: *const u32,
    pub table_stride: u64,
    pub offsets: *const u32,
    pub first: *const u32,
    pub n_seqs: u32,
    pub max_pages: u32,
    pub page_rows: u32,
}
#[repr(C)]
pub struct agpu_state {
    pub src: *const c_void,
    pub dst: *mut c_void,
    pub src_row_stride: u64,
    pub src_piece_stride: u64,
    pub dst_row_stride: u64,
    pub dst_piece_stride: u64,
    pub n_pieces: u64,
    pub piece_bytes: u64,
    pub position_bytes: u64,
}
#[repr(C)]
pub struct agpu_beams {
    pub logits: *const c_void,
    pub row_stride: u64,
    pub row_type: i32,
    pub batch: u32,
    pub beams: u32,
    pub vocab: u32,
    pub k: u32,
    pub end_token: u32,
    pub scores: *const f32,
    pub allowed: *const c_void,
    pub allowed_stride: u64,
    pub finished: *const c_void,
    pub out_scores: *mut f32,
    pub out_parents: *mut u32,
    pub out_tokens: *mut u32,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
}
#[repr(C)]
pub struct agpu_comm_peer {
    pub rank: i32,
    pub world: i32,
    pub device_ordinal: i32,
    pub nccl_device: i32,
    pub pci_domain: i32,
    pub pci_bus: i32,
    pub pci_device: i32,
    pub pid: i32,
    pub host_hash: u64,
    pub uuid: [u8; 16],
    pub gcn_arch: [c_char; 16],
}
#[repr(C)]
pub struct ArrowSchema {
    pub format: *const c_char,
    pub name: *const c_char,
    pub metadata: *const c_char,
    pub flags: i64,
    pub n_children: i64,
    pub children: *mut *mut ArrowSchema,
    pub dictionary: *mut ArrowSchema,
    pub release: Option<unsafe extern "C" fn(*mut ArrowSchema)>,
    pub private_data: *mut c_void,
}
#[repr(C)]
pub struct ArrowArray {
    pub length: i64,
    pub null_count: i64,
    pub offset: i64,
    pub n_buffers: i64,
    pub n_children: i64,
    pub buffers: *mut *const c_void,
    pub children: *mut *mut ArrowArray,
    pub dictionary: *mut ArrowArray,
    pub release: Option<unsafe extern "C" fn(*mut ArrowArray)>,
    pub private_data: *mut c_void,
}
#[repr(C)]
pub struct ArrowArrayStream {
    pub get_schema: Option<unsafe extern "C" fn(*mut ArrowArrayStream, *mut ArrowSchema) -> c_int>,
    pub get_next: Option<unsafe extern "C" fn(*mut ArrowArrayStream, *mut ArrowArray) -> c_int>,
    pub get_last_error: Option<unsafe extern "C" fn(*mut ArrowArrayStream) -> *const c_char>,
    pub release: Option<unsafe extern "C" fn(*mut ArrowArrayStream)>,
    pub private_data: *mut c_void,
}
#[repr(C)]
pub struct agpu_arrow_column {
    pub dtype: agpu_dtype,
    pub length: u64,
    pub null_count: i64,
    pub values: *mut c_void,
    pub validity: *mut c_void,
    pub values_bytes: u64,
    pub validity_bytes: u64,
}
#[repr(C)]
pub struct agpu_ipc_field {
    pub name: *const c_char,
    pub format: *const c_char,
    pub dtype: i32,
    pub nullable: i32,
}

#[link(name = "arrow_gpu_hip")]
extern "C" {
    pub fn agpu_abi_version() -> i32;
    pub fn agpu_last_error() -> *const c_char;
    pub fn agpu_build_info() -> *const c_char;
    pub fn agpu_dtype_size(t: agpu_dtype) -> usize;
    pub fn agpu_bitmap_bytes(n_bits: u64) -> usize;
    pub fn agpu_device_count(out_count: *mut i32) -> agpu_status;
    pub fn agpu_device_create(ordinal: i32, out_device: *mut *mut agpu_device) -> agpu_status;
    pub fn agpu_device_destroy(dev: *mut agpu_device) -> agpu_status;
    pub fn agpu_device_sync(dev: *mut agpu_device) -> agpu_status;
    pub fn agpu_device_download(dev: *mut agpu_device, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_device_name(dev: *mut agpu_device, out: *mut c_char, out_cap: usize) -> agpu_status;
    pub fn agpu_device_ordinal(dev: *mut agpu_device, out_ordinal: *mut i32) -> agpu_status;
    pub fn agpu_device_mem_info(dev: *mut agpu_device, out_free: *mut u64, out_total: *mut u64) -> agpu_status;
    pub fn agpu_device_trim(dev: *mut agpu_device) -> agpu_status;
    pub fn agpu_device_pool_info(dev: *mut agpu_device, out_cached_bytes: *mut u64, out_cached_blocks: *mut u64, out_idle_streams: *mut u64) -> agpu_status;
    pub fn agpu_device_small_pool_info(dev: *mut agpu_device, out_slab_bytes: *mut u64, out_free_blocks: *mut u64, out_live_blocks: *mut u64) -> agpu_status;
    pub fn agpu_malloc(dev: *mut agpu_device, bytes: usize, zero_fill: i32, out_ptr: *mut *mut c_void) -> agpu_status;
    pub fn agpu_free(dev: *mut agpu_device, ptr: *mut c_void) -> agpu_status;
    pub fn agpu_malloc_like(dev: *mut agpu_device, bytes: usize, zero_fill: i32, neighbours: *const *const c_void, n_neighbours: i32, out_ptr: *mut *mut c_void) -> agpu_status;
    pub fn agpu_malloc_table(dev: *mut agpu_device, n_columns: i32, bytes: *const u64, zero_fill: i32, out_ptrs: *mut *mut c_void) -> agpu_status;
    pub fn agpu_upload(p: *mut agpu_pipeline, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_download(p: *mut agpu_pipeline, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_copy(p: *mut agpu_pipeline, dst_dev: *mut c_void, src_dev: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_memset(p: *mut agpu_pipeline, dst_dev: *mut c_void, byte_value: i32, bytes: usize) -> agpu_status;
    pub fn agpu_host_alloc(dev: *mut agpu_device, bytes: usize, out_host_ptr: *mut *mut c_void) -> agpu_status;
    pub fn agpu_host_free(dev: *mut agpu_device, host_ptr: *mut c_void) -> agpu_status;
    pub fn agpu_upload_async(p: *mut agpu_pipeline, dst_dev: *mut c_void, src_pinned: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_download_async(p: *mut agpu_pipeline, dst_pinned: *mut c_void, src_dev: *const c_void, bytes: usize) -> agpu_status;
    pub fn agpu_pipeline_create(dev: *mut agpu_device, out_pipeline: *mut *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_wrap_stream(dev: *mut agpu_device, hip_stream: *mut c_void, out_pipeline: *mut *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_finish(p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_sync(p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_destroy(p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_device(p: *mut agpu_pipeline, out_device: *mut *mut agpu_device) -> agpu_status;
    pub fn agpu_pipeline_stream(p: *mut agpu_pipeline, out_hip_stream: *mut *mut c_void) -> agpu_status;
    pub fn agpu_pipeline_wait_pipeline(p: *mut agpu_pipeline, other: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_begin_capture(p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_pipeline_end_capture(p: *mut agpu_pipeline, out_graph: *mut *mut agpu_graph) -> agpu_status;
    pub fn agpu_graph_launch(g: *mut agpu_graph, p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_graph_destroy(g: *mut agpu_graph) -> agpu_status;
    pub fn agpu_event_create(dev: *mut agpu_device, out_event: *mut *mut agpu_event) -> agpu_status;
    pub fn agpu_event_record(e: *mut agpu_event, p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_event_elapsed_ms(start: *mut agpu_event, stop: *mut agpu_event, out_ms: *mut f32) -> agpu_status;
    pub fn agpu_event_destroy(e: *mut agpu_event) -> agpu_status;
    pub fn agpu_pipeline_enable_timing(p: *mut agpu_pipeline, profile_bits: i32) -> agpu_status;
    pub fn agpu_pipeline_last_kernel_ns(p: *mut agpu_pipeline, out_ns: *mut u64, out_name: *mut *const c_char) -> agpu_status;
    pub fn agpu_set_tuning(key: *const c_char, value: i64) -> agpu_status;
    pub fn agpu_get_tuning(key: *const c_char, out_value: *mut i64) -> agpu_status;
    pub fn agpu_pipeline_set_tuning(p: *mut agpu_pipeline, key: *const c_char, value: i64) -> agpu_status;
    pub fn agpu_pipeline_get_tuning(p: *mut agpu_pipeline, key: *const c_char, out_value: *mut i64) -> agpu_status;
    pub fn agpu_binary(p: *mut agpu_pipeline, op: agpu_binary_op, dtype: agpu_dtype, a: *const c_void, b: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_scalar(p: *mut agpu_pipeline, op: agpu_binary_op, dtype: agpu_dtype, a: *const c_void, scalar: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_unary(p: *mut agpu_pipeline, op: agpu_unary_op, dtype: agpu_dtype, r#in: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_selftest_unary_f32(p: *mut agpu_pipeline, op: agpu_unary_op, first_bits: u64, count: u64, out_max_ulp: *mut u32, out_worst_bits: *mut u32) -> agpu_status;
    pub fn agpu_selftest_pow_f32(p: *mut agpu_pipeline, seed: u64, count: u64, domain: i32, out_max_ulp: *mut u32, out_worst_x_bits: *mut u32, out_worst_y_bits: *mut u32) -> agpu_status;
    pub fn agpu_cast(p: *mut agpu_pipeline, from: agpu_dtype, to: agpu_dtype, r#in: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_broadcast(p: *mut agpu_pipeline, dtype: agpu_dtype, value_bits: u32, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_broadcast_from_device(p: *mut agpu_pipeline, dtype: agpu_dtype, scalar_dev: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_fused_chain(p: *mut agpu_pipeline, dtype: agpu_dtype, r#in: *const c_void, steps: *const agpu_chain_step, n_steps: i32, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_fused_chain_compare(p: *mut agpu_pipeline, dtype: agpu_dtype, r#in: *const c_void, steps: *const agpu_chain_step, n_steps: i32, cmp_op: agpu_cmp_op, operand_kind: i32, operand: *const c_void, out_bits: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_fused_cast_chain(p: *mut agpu_pipeline, from: agpu_dtype, r#in: *const c_void, steps: *const agpu_chain_step, n_steps: i32, out: *mut f32, n: u64) -> agpu_status;
    pub fn agpu_compare(p: *mut agpu_pipeline, op: agpu_cmp_op, dtype: agpu_dtype, a: *const c_void, b: *const c_void, out_bits: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_compare_validity(p: *mut agpu_pipeline, op: agpu_cmp_op, dtype: agpu_dtype, a: *const c_void, b: *const c_void, va: *const c_void, vb: *const c_void, out_bits: *mut c_void, out_validity: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_compare_validity_count(p: *mut agpu_pipeline, op: agpu_cmp_op, dtype: agpu_dtype, a: *const c_void, b: *const c_void, va: *const c_void, vb: *const c_void, out_bits: *mut c_void, out_validity: *mut c_void, n: u64, out_null_count_dev: *mut u64) -> agpu_status;
    pub fn agpu_bitmap_binary(p: *mut agpu_pipeline, op: agpu_binary_op, a: *const c_void, b: *const c_void, out: *mut c_void, n_bits: u64) -> agpu_status;
    pub fn agpu_bitmap_binary_count(p: *mut agpu_pipeline, op: agpu_binary_op, a: *const c_void, b: *const c_void, out: *mut c_void, n_bits: u64, out_set_count_dev: *mut u64) -> agpu_status;
    pub fn agpu_bitmap_not(p: *mut agpu_pipeline, r#in: *const c_void, out: *mut c_void, n_bits: u64) -> agpu_status;
    pub fn agpu_bitmap_popcount(p: *mut agpu_pipeline, bits: *const c_void, n_bits: u64, out_count_dev: *mut u64) -> agpu_status;
    pub fn agpu_bitmap_any(p: *mut agpu_pipeline, bits: *const c_void, n_bits: u64, out_any_dev: *mut u32) -> agpu_status;
    pub fn agpu_bitmap_copy_bits(p: *mut agpu_pipeline, src: *const c_void, src_bit_offset: u64, out: *mut c_void, n_bits: u64) -> agpu_status;
    pub fn agpu_bitmap_merge_validity(p: *mut agpu_pipeline, va: *const c_void, vb: *const c_void, mask: *const c_void, vmask: *const c_void, out: *mut c_void, n_bits: u64) -> agpu_status;
    pub fn agpu_bitmap_merge_validity_count(p: *mut agpu_pipeline, va: *const c_void, vb: *const c_void, mask: *const c_void, vmask: *const c_void, out: *mut c_void, n_bits: u64, out_set_count_dev: *mut u64) -> agpu_status;
    pub fn agpu_reduce(p: *mut agpu_pipeline, op: agpu_reduce_op, dtype: agpu_dtype, r#in: *const c_void, validity: *const c_void, n: u64, out_dev: *mut c_void) -> agpu_status;
    pub fn agpu_reduce_sum_f64(p: *mut agpu_pipeline, r#in: *const f32, validity: *const c_void, n: u64, out_dev: *mut f64) -> agpu_status;
    pub fn agpu_reduce_stats_f32(p: *mut agpu_pipeline, r#in: *const f32, validity: *const c_void, n: u64, out_dev: *mut agpu_f32_stats) -> agpu_status;
    pub fn agpu_take(p: *mut agpu_pipeline, width: i32, values: *const c_void, n_values: u64, idx: *const u32, out: *mut c_void, n_idx: u64) -> agpu_status;
    pub fn agpu_take_columns(p: *mut agpu_pipeline, n_cols: i32, widths: *const i32, values: *const *const c_void, n_values: u64, idx: *const u32, outs: *const *mut c_void, n_idx: u64) -> agpu_status;
    pub fn agpu_take_columns_validity(p: *mut agpu_pipeline, n_cols: i32, widths: *const i32, values: *const *const c_void, validities: *const *const c_void, n_values: u64, idx: *const u32, outs: *const *mut c_void, out_validities: *const *mut c_void, n_idx: u64) -> agpu_status;
    pub fn agpu_take_validity(p: *mut agpu_pipeline, width: i32, values: *const c_void, n_values: u64, validity: *const c_void, idx: *const u32, out: *mut c_void, out_validity: *mut c_void, n_idx: u64) -> agpu_status;
    pub fn agpu_take_bits(p: *mut agpu_pipeline, bits: *const c_void, n_bits: u64, idx: *const u32, out_bits: *mut c_void, n_idx: u64) -> agpu_status;
    pub fn agpu_put_bounded(p: *mut agpu_pipeline, width: i32, src: *const c_void, n_src: u64, src_idx: *const u32, dst: *mut c_void, n_dst: u64, dst_idx: *const u32, n: u64) -> agpu_status;
    pub fn agpu_put(p: *mut agpu_pipeline, width: i32, src: *const c_void, src_idx: *const u32, dst: *mut c_void, dst_idx: *const u32, n: u64) -> agpu_status;
    pub fn agpu_put_bits_bounded(p: *mut agpu_pipeline, src_bits: *const c_void, n_src_bits: u64, src_idx: *const u32, dst_bits: *mut c_void, n_dst_bits: u64, dst_idx: *const u32, n: u64) -> agpu_status;
    pub fn agpu_put_bits(p: *mut agpu_pipeline, src_bits: *const c_void, src_idx: *const u32, dst_bits: *mut c_void, dst_idx: *const u32, n: u64) -> agpu_status;
    pub fn agpu_merge(p: *mut agpu_pipeline, width: i32, a: *const c_void, b: *const c_void, mask_bits: *const c_void, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_merge_bits(p: *mut agpu_pipeline, a: *const c_void, b: *const c_void, mask_bits: *const c_void, out: *mut c_void, n_bits: u64) -> agpu_status;
    pub fn agpu_index_max(p: *mut agpu_pipeline, idx: *const u32, n: u64, out_max_dev: *mut u32) -> agpu_status;
    pub fn agpu_put_quantised(p: *mut agpu_pipeline, n_cols: i32, stores: *const agpu_quantised_rows, rows: *const agpu_rows, slots: *const u32, n: u64) -> agpu_status;
    pub fn agpu_put_quantised_pages(p: *mut agpu_pipeline, n_cols: i32, stores: *const agpu_quantised_rows, rows: *const agpu_rows, pages: *const agpu_page_map, n: u64) -> agpu_status;
    pub fn agpu_take_quantised(p: *mut agpu_pipeline, n_cols: i32, stores: *const agpu_quantised_rows, rows: *const agpu_rows, slots: *const u32, n: u64) -> agpu_status;
    pub fn agpu_take_quantised_pages(p: *mut agpu_pipeline, n_cols: i32, stores: *const agpu_quantised_rows, rows: *const agpu_rows, pages: *const agpu_page_map, n: u64) -> agpu_status;
    pub fn agpu_take_rows(p: *mut agpu_pipeline, n_states: i32, states: *const agpu_state, n_src: u64, idx: *const u32, lengths: *const u32, n: u64) -> agpu_status;
    pub fn agpu_select_beams_workspace(batch: u32, beams: u32, vocab: u32, k: u32, out_bytes: *mut u64) -> agpu_status;
    pub fn agpu_select_beams(p: *mut agpu_pipeline, args: *const agpu_beams) -> agpu_status;
    pub fn agpu_comm_get_unique_id(out_id: *mut c_void) -> agpu_status;
    pub fn agpu_comm_init_rank(dev: *mut agpu_device, unique_id: *const c_void, rank: i32, world: i32, out_comm: *mut *mut agpu_comm) -> agpu_status;
    pub fn agpu_comm_init_rank_timeout(dev: *mut agpu_device, unique_id: *const c_void, rank: i32, world: i32, timeout_ms: i64, out_comm: *mut *mut agpu_comm) -> agpu_status;
    pub fn agpu_comm_runtime_info(out: *mut c_char, out_cap: usize) -> agpu_status;
    pub fn agpu_comm_destroy(c: *mut agpu_comm) -> agpu_status;
    pub fn agpu_comm_rank(c: *mut agpu_comm, out_rank: *mut i32, out_world: *mut i32) -> agpu_status;
    pub fn agpu_comm_reduce(c: *mut agpu_comm, p: *mut agpu_pipeline, op: agpu_reduce_op, dtype: agpu_dtype, r#in: *const c_void, validity: *const c_void, n_local: u64, out_dev: *mut c_void) -> agpu_status;
    pub fn agpu_comm_reduce_sum_f64(c: *mut agpu_comm, p: *mut agpu_pipeline, r#in: *const f32, validity: *const c_void, n_local: u64, out_dev: *mut f64) -> agpu_status;
    pub fn agpu_comm_reduce_stats_f32(c: *mut agpu_comm, p: *mut agpu_pipeline, r#in: *const f32, validity: *const c_void, n_local: u64, out_dev: *mut agpu_f32_stats) -> agpu_status;
    pub fn agpu_comm_final_reduce(c: *mut agpu_comm, p: *mut agpu_pipeline, op: agpu_reduce_op, dtype: agpu_dtype, kind_f64: i32, partial_dev: *const c_void, n_local: u64, out_dev: *mut c_void) -> agpu_status;
    pub fn agpu_reduce_combine(p: *mut agpu_pipeline, op: agpu_reduce_op, dtype: agpu_dtype, kind_f64: i32, records_dev: *const c_void, world: i32, out_dev: *mut c_void) -> agpu_status;
    pub fn agpu_comm_all_reduce(c: *mut agpu_comm, p: *mut agpu_pipeline, op: agpu_reduce_op, ctype: agpu_comm_dtype, buf_dev: *mut c_void, count: u64) -> agpu_status;
    pub fn agpu_comm_barrier(c: *mut agpu_comm, p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_comm_sync(c: *mut agpu_comm, p: *mut agpu_pipeline) -> agpu_status;
    pub fn agpu_comm_size(c: *mut agpu_comm, out_count: *mut i32, out_user_rank: *mut i32, out_device: *mut i32) -> agpu_status;
    pub fn agpu_comm_is_local(c: *mut agpu_comm, out_local: *mut i32) -> agpu_status;
    pub fn agpu_device_identity(dev: *mut agpu_device, out: *mut agpu_comm_peer) -> agpu_status;
    pub fn agpu_comm_peers(c: *mut agpu_comm, p: *mut agpu_pipeline, out_host: *mut agpu_comm_peer, cap: i32, out_distinct: *mut i32) -> agpu_status;
    pub fn agpu_import_arrow(p: *mut agpu_pipeline, array: *const ArrowArray, schema: *const ArrowSchema, out_column: *mut agpu_arrow_column) -> agpu_status;
    pub fn agpu_import_arrow_table(p: *mut agpu_pipeline, n_columns: i32, arrays: *const *const ArrowArray, schemas: *const *const ArrowSchema, out_columns: *mut agpu_arrow_column) -> agpu_status;
    pub fn agpu_import_arrow_stream_next(p: *mut agpu_pipeline, stream: *mut ArrowArrayStream, columns: *const i32, n_columns: i32, out_columns: *mut agpu_arrow_column, out_rows: *mut i64) -> agpu_status;
    pub fn agpu_export_arrow(p: *mut agpu_pipeline, column: *const agpu_arrow_column, out_array: *mut ArrowArray, out_schema: *mut ArrowSchema) -> agpu_status;
    pub fn agpu_arrow_column_free(dev: *mut agpu_device, column: *mut agpu_arrow_column) -> agpu_status;
    pub fn agpu_staged_copy(p: *mut agpu_pipeline, dev_ptr: *mut c_void, host_ptr: *mut c_void, bytes: usize, to_device: i32) -> agpu_status;
    pub fn agpu_ipc_open(data: *const c_void, bytes: u64, out_reader: *mut *mut agpu_ipc_reader) -> agpu_status;
    pub fn agpu_ipc_close(r: *mut agpu_ipc_reader);
    pub fn agpu_ipc_num_fields(r: *const agpu_ipc_reader, out_n: *mut i32) -> agpu_status;
    pub fn agpu_ipc_field_info(r: *const agpu_ipc_reader, i: i32, out: *mut agpu_ipc_field) -> agpu_status;
    pub fn agpu_ipc_num_batches(r: *const agpu_ipc_reader, out_n: *mut i64) -> agpu_status;
    pub fn agpu_ipc_batch_rows(r: *const agpu_ipc_reader, batch: i64, out_rows: *mut i64) -> agpu_status;
    pub fn agpu_ipc_column_view(r: *const agpu_ipc_reader, batch: i64, column: i32, out_array: *mut ArrowArray, out_schema: *mut ArrowSchema) -> agpu_status;
    pub fn agpu_ipc_read_column(r: *const agpu_ipc_reader, batch: i64, column: i32, p: *mut agpu_pipeline, out_column: *mut agpu_arrow_column) -> agpu_status;
    pub fn agpu_ipc_read_batch(r: *const agpu_ipc_reader, batch: i64, columns: *const i32, n_columns: i32, p: *mut agpu_pipeline, out_columns: *mut agpu_arrow_column) -> agpu_status;
    pub fn agpu_ipc_writer_create(fields: *const agpu_ipc_field, n_fields: i32, file_format: i32, fd: i32, out_writer: *mut *mut agpu_ipc_writer) -> agpu_status;
    pub fn agpu_ipc_writer_set_compression(w: *mut agpu_ipc_writer, codec: i32) -> agpu_status;
    pub fn agpu_ipc_writer_write_batch(w: *mut agpu_ipc_writer, columns: *const *const ArrowArray) -> agpu_status;
    pub fn agpu_ipc_writer_write_device_batch(w: *mut agpu_ipc_writer, p: *mut agpu_pipeline, columns: *const agpu_arrow_column) -> agpu_status;
    pub fn agpu_ipc_writer_finish(w: *mut agpu_ipc_writer, out_data: *mut *const c_void, out_bytes: *mut u64) -> agpu_status;
    pub fn agpu_ipc_writer_destroy(w: *mut agpu_ipc_writer);
    pub fn agpu_launch_by_name(p: *mut agpu_pipeline, shader_key: *const c_char, entry_point: *const c_char, inputs: *const *const c_void, n_inputs: i32, out: *mut c_void, n: u64) -> agpu_status;
    pub fn agpu_shader_key_for_source(wgsl: *const c_char, len: usize, out_key: *mut c_char, out_cap: usize) -> agpu_status;
    pub fn agpu_shader_key_for_hash(fnv1a64_of_text: u64, text_bytes: u64, out_key: *mut c_char, out_cap: usize) -> agpu_status;
    pub fn agpu_launch_by_name_sized(p: *mut agpu_pipeline, shader_key: *const c_char, entry_point: *const c_char, inputs: *const *const c_void, input_bytes: *const u64, n_inputs: i32, out: *mut c_void, out_bytes: u64, dispatch_size: u32) -> agpu_status;
    pub fn agpu_synth_f32(p: *mut agpu_pipeline, out: *mut f32, n: u64, seed: u64, row0: u64, lo: f32, hi: f32) -> agpu_status;
    pub fn agpu_synth_i32(p: *mut agpu_pipeline, out: *mut i32, n: u64, seed: u64, row0: u64, modulus: u32) -> agpu_status;
    pub fn agpu_synth_u8(p: *mut agpu_pipeline, out: *mut u8, n: u64, seed: u64, row0: u64) -> agpu_status;
    pub fn agpu_synth_bits(p: *mut agpu_pipeline, out_bits: *mut c_void, n_bits: u64, seed: u64, row0: u64, p_set: f64) -> agpu_status;
    pub fn agpu_checksum(p: *mut agpu_pipeline, data: *const c_void, bytes: u64, out_sum_dev: *mut u64) -> agpu_status;
}
