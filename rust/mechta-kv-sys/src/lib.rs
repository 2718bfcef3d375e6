//! Raw bindings of libmechta_kv (include/mechta_kv.h), the C ABI of the B200 KV-cache / attention path.
//!
//! GENERATED by gen_bindings.py from the header; do not edit by hand. NOT COMPILED where it was written (no Rust
//! toolchain there): names, argument counts and types are checked textually against the header by the test suite.
//! This crate is the one `unsafe` surface of the path, as engine/crates/shader is in the reference; the safe
//! wrapper is the `mechta-kv` crate beside it. Link with `-lmechta_kv` (see build.rs).
#![allow(non_camel_case_types)]

use core::ffi::{c_char, c_int, c_void};

pub type mkv_status = c_int;
pub type mkv_fmt = c_int;
pub const MKV_OK: mkv_status = 0;
pub const MKV_ERR_INVALID: mkv_status = 1;
pub const MKV_ERR_CAPACITY: mkv_status = 2;
pub const MKV_ERR_CUDA: mkv_status = 3;
pub const MKV_ERR_NOMEM: mkv_status = 4;
pub const MKV_ERR_UNSUPPORTED: mkv_status = 5;
pub const MKV_ERR_STATE: mkv_status = 6;
pub const MKV_ERR_FORMAT: mkv_status = 7;
pub const MKV_ERR_IO: mkv_status = 8;
pub const MKV_F16: mkv_fmt = 0;
pub const MKV_F32: mkv_fmt = 1;
pub const MKV_HQ: c_int = 16;
pub const MKV_HKV: c_int = 2;
pub const MKV_D: c_int = 256;
pub const MKV_GROUP: c_int = 8;
pub const MKV_ROW: c_int = 512;
pub const MKV_MAX_VERIFY: c_int = 4;
pub const MKV_REC: c_int = 258;
pub const MKV_CTX_MIN: c_int = 4096;
pub const MKV_CTX_MAX: c_int = 262144;
pub const MKV_ROPE_HALF: c_int = 0;
pub const MKV_ROPE_INTERLEAVED: c_int = 1;
pub const MKV_SCALE_NONE: c_int = 0;
pub const MKV_SCALE_LINEAR: c_int = 1;
pub const MKV_SCALE_NTK: c_int = 2;
pub const MKV_SCALE_YARN: c_int = 3;
pub const MKV_ROPE_MAX_DIMS: c_int = 256;

#[repr(C)]
pub struct mkv_ctx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct mkv_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct mkv_exchange {
    _private: [u8; 0],
}
#[repr(C)]
pub struct mkv_rope {
    _private: [u8; 0],
}
#[repr(C)]
pub struct mkv_pool {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_verify_item {
    pub cache: *mut mkv_cache,
    pub layer: i32,
    pub first_pos: u32,
    pub pos: u32,
    pub ntok: u32,
    pub q_dev: *const f32,
    pub out_dev: *mut f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_step_in {
    pub qf_dev: *const f32,
    pub kb_dev: *const f32,
    pub vb_dev: *const f32,
    pub q_norm_dev: *const f32,
    pub k_norm_dev: *const f32,
    pub rope_tab_dev: *const f32,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_rope_desc {
    pub dims: i32,
    pub layout: i32,
    pub scaling: i32,
    pub base: f64,
    pub factor: f64,
    pub original: f64,
    pub slow: f64,
    pub fast: f64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_rope_rows {
    pub x_dev: *const c_void,
    pub y_dev: *mut c_void,
    pub x_fmt: mkv_fmt,
    pub y_fmt: mkv_fmt,
    pub ntok: u32,
    pub heads: u32,
    pub head_dim: u32,
    pub x_token_stride: i64,
    pub x_head_stride: i64,
    pub y_token_stride: i64,
    pub y_head_stride: i64,
    pub pos_dev: *const i32,
    pub backward: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_pool_desc {
    pub fmt: mkv_fmt,
    pub n_layers: i32,
    pub n_pages: u32,
    pub page_tokens: u32,
    pub max_seqs: u32,
    pub max_tokens: u32,
    pub q_heads: i32,
    pub kv_heads: i32,
    pub head_dim: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_seq_rows {
    pub seq: u32,
    pub first_pos: u32,
    pub pos: u32,
    pub ntok: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_pool_rows {
    pub k_dev: *const c_void,
    pub v_dev: *const c_void,
    pub fmt: mkv_fmt,
    pub k_stride: i64,
    pub v_stride: i64,
    pub rope: *const mkv_rope,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mkv_pool_attn {
    pub q_dev: *const c_void,
    pub out_dev: *mut c_void,
    pub q_stride: i64,
    pub out_stride: i64,
    pub scale: f32,
    pub window: u32,
    pub sinks_dev: *const f32,
}

extern "C" {
    pub fn mkv_strerror(s: mkv_status) -> *const c_char;
    pub fn mkv_last_error() -> *const c_char;
    pub fn mkv_version() -> *const c_char;
    pub fn mkv_ctx_create(device: c_int, stream: *mut c_void, out: *mut *mut mkv_ctx) -> mkv_status;
    pub fn mkv_ctx_destroy(ctx: *mut mkv_ctx);
    pub fn mkv_sync(ctx: *mut mkv_ctx) -> mkv_status;
    pub fn mkv_launch_count(ctx: *const mkv_ctx) -> u64;
    pub fn mkv_prof_enable(ctx: *mut mkv_ctx, on: c_int) -> mkv_status;
    pub fn mkv_prof_read(ctx: *mut mkv_ctx, core_ms: *mut f64, core_launches: *mut u64) -> mkv_status;
    pub fn mkv_cache_create(ctx: *mut mkv_ctx, fmt: mkv_fmt, n_layers: c_int, context_tokens: u32, shard_first: u32, shard_tokens: u32, out: *mut *mut mkv_cache) -> mkv_status;
    pub fn mkv_cache_destroy(c: *mut mkv_cache);
    pub fn mkv_cache_buffers(c: *mut mkv_cache, layer: c_int, k_dev: *mut *mut c_void, v_dev: *mut *mut c_void) -> mkv_status;
    pub fn mkv_cache_len(c: *const mkv_cache) -> u32;
    pub fn mkv_cache_set_len(c: *mut mkv_cache, len: u32) -> mkv_status;
    pub fn mkv_need_bytes(ctx_tokens: u32, fmt: mkv_fmt, n_layers: c_int) -> u64;
    pub fn mkv_cache_device_bytes(c: *const mkv_cache) -> u64;
    pub fn mkv_append(c: *mut mkv_cache, layer: c_int, pos: u32, ntok: u32, k_dev: *const f32, v_dev: *const f32, rope_tab_dev: *const f32) -> mkv_status;
    pub fn mkv_append_layers(c: *mut mkv_cache, pos: u32, ntok: u32, k_dev: *const f32, v_dev: *const f32, rope_tab_dev: *const f32) -> mkv_status;
    pub fn mkv_rope_table(pos: i32, ntok: u32, out_host: *mut f32);
    pub fn mkv_truncate(c: *mut mkv_cache, new_len: u32, scrub: c_int) -> mkv_status;
    pub fn mkv_attn_verify(c: *mut mkv_cache, layer: c_int, first_pos: u32, pos: u32, ntok: u32, q_dev: *const f32, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_attn_verify_partial(c: *mut mkv_cache, layer: c_int, first_pos: u32, pos: u32, ntok: u32, q_dev: *const f32, rec_dev: *mut f32) -> mkv_status;
    pub fn mkv_combine_shards(ctx: *mut mkv_ctx, recs_dev: *const f32, n_shards: c_int, ntok: u32, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_exchange_create(ctx: *mut mkv_ctx, rank: c_int, world: c_int, out: *mut *mut mkv_exchange) -> mkv_status;
    pub fn mkv_exchange_handle(ex: *mut mkv_exchange, handle_out_64_bytes: *mut c_void) -> mkv_status;
    pub fn mkv_exchange_connect(ex: *mut mkv_exchange, handles: *const c_void) -> mkv_status;
    pub fn mkv_exchange_destroy(ex: *mut mkv_exchange);
    pub fn mkv_attn_verify_exchange(c: *mut mkv_cache, ex: *mut mkv_exchange, layer: c_int, first_pos: u32, pos: u32, ntok: u32, q_dev: *const f32, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_attn_verify_static(device: c_int, stream: *mut c_void, k_dev: *const c_void, v_dev: *const c_void, capacity_tokens: u32, first_pos: u32, pos: u32, ntok: u32, q_dev: *const f32, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_static_status(device: c_int, stream: *mut c_void, status_out: *mut u32) -> mkv_status;
    pub fn mkv_attn_verify_batch(ctx: *mut mkv_ctx, items: *const mkv_verify_item, n: c_int) -> mkv_status;
    pub fn mkv_cache_create_ring(ctx: *mut mkv_ctx, fmt: mkv_fmt, n_layers: c_int, context_tokens: u32, ring_rows: u32, out: *mut *mut mkv_cache) -> mkv_status;
    pub fn mkv_attn_verify_window(c: *mut mkv_cache, layer: c_int, window: u32, sinks_dev: *const f32, pos: u32, ntok: u32, q_dev: *const f32, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_attn_step(c: *mut mkv_cache, layer: c_int, first_pos: u32, pos: u32, ntok: u32, r#in: *const mkv_step_in, ag_dev: *mut f32, ag16_dev: *mut c_void) -> mkv_status;
    pub fn mkv_attn_prefill(c: *mut mkv_cache, layer: c_int, first_pos: u32, pos0: u32, ntok: u32, q_dev: *const c_void, q_is_f16: c_int, out_dev: *mut f32) -> mkv_status;
    pub fn mkv_rope_create(desc: *const mkv_rope_desc, out: *mut *mut mkv_rope) -> mkv_status;
    pub fn mkv_rope_destroy(r: *mut mkv_rope);
    pub fn mkv_rope_freqs(r: *const mkv_rope, freqs_host: *mut f64, m_host: *mut f64) -> mkv_status;
    pub fn mkv_rope_apply(ctx: *mut mkv_ctx, r: *const mkv_rope, rows: *const mkv_rope_rows) -> mkv_status;
    pub fn mkv_pool_create(ctx: *mut mkv_ctx, desc: *const mkv_pool_desc, out: *mut *mut mkv_pool) -> mkv_status;
    pub fn mkv_pool_destroy(p: *mut mkv_pool);
    pub fn mkv_pool_buffers(p: *mut mkv_pool, layer: c_int, k_dev: *mut *mut c_void, v_dev: *mut *mut c_void) -> mkv_status;
    pub fn mkv_pool_free_pages(p: *const mkv_pool) -> u32;
    pub fn mkv_seq_create(p: *mut mkv_pool, seq_out: *mut u32) -> mkv_status;
    pub fn mkv_seq_fork(p: *mut mkv_pool, seq: u32, len: u32, copy: c_int, n: c_int, children_host: *mut u32) -> mkv_status;
    pub fn mkv_seq_free(p: *mut mkv_pool, seqs_host: *const u32, n: c_int) -> mkv_status;
    pub fn mkv_seq_truncate(p: *mut mkv_pool, seq: u32, len: u32) -> mkv_status;
    pub fn mkv_seq_set_len(p: *mut mkv_pool, seq: u32, len: u32) -> mkv_status;
    pub fn mkv_seq_len(p: *const mkv_pool, seq: u32) -> u32;
    pub fn mkv_seq_pages(p: *const mkv_pool, seq: u32, pages_host: *mut u32, cap: u32, n_out: *mut u32) -> mkv_status;
    pub fn mkv_pool_compact(p: *mut mkv_pool, moved_out: *mut u32) -> mkv_status;
    pub fn mkv_pool_write(p: *mut mkv_pool, layer: c_int, items: *const mkv_seq_rows, n: c_int, r#in: *const mkv_pool_rows) -> mkv_status;
    pub fn mkv_attn_pool(p: *mut mkv_pool, layer: c_int, items: *const mkv_seq_rows, n: c_int, r#in: *const mkv_pool_attn) -> mkv_status;
    pub fn mkv_snapshot_bytes(c: *const mkv_cache, p: u32) -> usize;
    pub fn mkv_snapshot(c: *mut mkv_cache, p: u32, dst_host: *mut c_void, cap: usize, written: *mut usize) -> mkv_status;
    pub fn mkv_snapshot_wait(c: *mut mkv_cache) -> mkv_status;
    pub fn mkv_restore(c: *mut mkv_cache, p: u32, src_host: *const c_void, bytes: usize) -> mkv_status;
    pub fn mkv_host_alloc(bytes: usize, out: *mut *mut c_void) -> mkv_status;
    pub fn mkv_host_free(p: *mut c_void);
    pub fn mkv_checks_enabled() -> c_int;
    pub fn mkv_cache_check_guards(c: *mut mkv_cache, bad_bytes: *mut u64) -> mkv_status;
    pub fn mkv_checks_touch_guard(c: *mut mkv_cache) -> mkv_status;
    pub fn mkv_root_write(path: *const c_char, fmt: mkv_fmt, n_layers: c_int, p: u32, tokens: *const u32, payload_host: *const c_void, payload_bytes: usize) -> mkv_status;
    pub fn mkv_root_read(path: *const c_char, fmt: mkv_fmt, n_layers: c_int, p_out: *mut u32, tokens_out: *mut u32, tokens_cap: usize, payload_host: *mut c_void, payload_cap: usize, payload_bytes: *mut usize) -> mkv_status;
    pub fn mkv_root_key(tokens: *const u32, n: usize) -> u64;
    pub fn mkv_dispatch(c: *mut mkv_cache, layer: c_int, op: *const c_char, u: *const u32, in0: *const c_void, in1: *const c_void, out: *mut c_void) -> mkv_status;
}
