//! Raw bindings of `include/bonsai_paged.h`: many requests over one paged KV cache held in 4 bits (rotary positions,
//! append, read-back, attention). The cache, the RoPE table and the activations are the caller's device memory.
//!
//! UNBUILT like the rest of the crate; kept in step with the header by `tests/test_paged_cpu.py`.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_int, c_void};

pub const BP_DTYPE_F16: u32 = 0;
pub const BP_DTYPE_BF16: u32 = 1;
pub const BP_ROPE_HALF: u32 = 0;
pub const BP_ROPE_INTERLEAVED: u32 = 1;
pub const BP_ROPE_SCALE_NONE: u32 = 0;
pub const BP_ROPE_SCALE_LINEAR: u32 = 1;
pub const BP_ROPE_SCALE_NTK: u32 = 2;
pub const BP_ROPE_SCALE_YARN: u32 = 3;

#[repr(C)]
pub struct bp_paged_ctx {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_rope_table {
    pub cos_sin: *const c_void,
    pub n_pos: u32,
    pub rot_dim: u32,
    pub layout: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_rope_config {
    pub n_pos: u32,
    pub rot_dim: u32,
    pub scaling: u32,
    pub freq_base: f32,
    pub factor: f32,
    pub beta_fast: f32,
    pub beta_slow: f32,
    pub orig_ctx: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_rows {
    pub data: *mut c_void,
    pub tok_stride: i64,
    pub head_stride: i64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_kv4_pool {
    pub data: *mut c_void,
    pub n_pages: u32,
    pub page_tokens: u32,
    pub n_kv_head: u32,
    pub head_dim: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_kv4_attn {
    pub q: bp_rows,
    pub out: bp_rows,
    pub q_start: *const c_void,
    pub kv_len: *const c_void,
    pub page_table: *const c_void,
    pub n_req: u32,
    pub n_head: u32,
    pub total_q: u32,
    pub max_q: u32,
    pub max_kv: u32,
    pub table_stride: u32,
    pub window: u32,
    pub scale: f32,
}

extern "C" {
    pub fn bp_paged_create(device: i32, out: *mut *mut bp_paged_ctx) -> c_int;
    pub fn bp_paged_destroy(ctx: *mut bp_paged_ctx);
    pub fn bp_paged_status(ctx: *mut bp_paged_ctx, stream: *mut c_void) -> c_int;
    pub fn bp_paged_last_error(ctx: *const bp_paged_ctx) -> *const c_char;
    pub fn bp_rope_fill(ctx: *mut bp_paged_ctx, stream: *mut c_void, cfg: *const bp_rope_config, table_out: *mut c_void) -> c_int;
    pub fn bp_rope(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, x: *const bp_rows, out: *const bp_rows, n_tok: u32, n_head: u32, head_dim: u32,
        positions: *const c_void, table: *const bp_rope_table, w_norm: *const c_void, eps: f32, inverse: u32,
    ) -> c_int;
    pub fn bp_kv4_pool_bytes(pool: *const bp_kv4_pool) -> u64;
    pub fn bp_kv4_append(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, k: *const bp_rows, v: *const bp_rows, n_tok: u32,
        positions: *const c_void, slots: *const c_void, table: *const bp_rope_table, w_k_norm: *const c_void, eps: f32,
    ) -> c_int;
    pub fn bp_kv4_read(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, slots: *const c_void, n_tok: u32, k: *const bp_rows,
        v: *const bp_rows,
    ) -> c_int;
    pub fn bp_kv4_attention(ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, args: *const bp_kv4_attn) -> c_int;
}
