//! Raw bindings of `include/bonsai_pages.h`: page tables on the device, attention behind a prefix in common, attention over chosen
//! pages. Everything but the context's scratch is the caller's device memory.
//!
//! UNBUILT like the rest of the crate; kept in step with the header by `tests/test_pages_cpu.py`.
#![allow(non_camel_case_types)]
use crate::paged::{bp_kv4_pool, bp_paged_ctx, bp_rows};
use std::os::raw::{c_int, c_void};

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_page_tables {
    pub table: *mut c_void,
    pub kv_len: *mut c_void,
    pub refs: *mut c_void,
    pub n_rows: u32,
    pub row_pages: u32,
    pub table_stride: u32,
    pub n_pages: u32,
    pub page_tokens: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_page_array {
    pub data: *mut c_void,
    pub page_bytes: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_kv4_shared {
    pub q: bp_rows,
    pub out: bp_rows,
    pub q_start: *const c_void,
    pub kv_len: *const c_void,
    pub page_table: *const c_void,
    pub prefix_start: *const c_void,
    pub prefix_len: *const c_void,
    pub prefix_table: *const c_void,
    pub work: *mut c_void,
    pub n_req: u32,
    pub n_head: u32,
    pub total_q: u32,
    pub max_q: u32,
    pub max_kv: u32,
    pub table_stride: u32,
    pub n_prefix: u32,
    pub max_prefix: u32,
    pub prefix_stride: u32,
    pub scale: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_block_summary {
    pub codes: *mut c_void,
    pub scales: *mut c_void,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_kv4_choice {
    pub q: bp_rows,
    pub q_start: *const c_void,
    pub kv_len: *const c_void,
    pub page_table: *const c_void,
    pub pages: *mut c_void,
    pub keys: *mut c_void,
    pub n_req: u32,
    pub n_head: u32,
    pub total_q: u32,
    pub max_q: u32,
    pub max_kv: u32,
    pub table_stride: u32,
    pub chosen: u32,
    pub first: u32,
    pub last: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct bp_kv4_chosen {
    pub q: bp_rows,
    pub out: bp_rows,
    pub pages: *const c_void,
    pub keys: *const c_void,
    pub n_head: u32,
    pub total_q: u32,
    pub chosen: u32,
    pub scale: f32,
}

extern "C" {
    pub fn bp_pages_grow(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, tables: *const bp_page_tables, n_new: *const c_void, q_start: *mut c_void,
        positions: *mut c_void, slots: *mut c_void, n_out: u32,
    ) -> c_int;
    pub fn bp_pages_release(ctx: *mut bp_paged_ctx, stream: *mut c_void, tables: *const bp_page_tables, rows: *const c_void, n: u32) -> c_int;
    pub fn bp_pages_fork(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, tables: *const bp_page_tables, parents: *const c_void, children: *const c_void, n: u32,
        src: *mut c_void, dst: *mut c_void,
    ) -> c_int;
    pub fn bp_pages_compact(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, tables: *const bp_page_tables, src: *mut c_void, dst: *mut c_void, most: u32,
    ) -> c_int;
    pub fn bp_pages_copy(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, arrays: *const bp_page_array, n_arrays: u32, n_pages: u32, src: *const c_void,
        dst: *const c_void, n: u32,
    ) -> c_int;
    pub fn bp_kv4_shared_work(total_q: u32, n_head: u32, head_dim: u32) -> u64;
    pub fn bp_kv4_attention_shared(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, args: *const bp_kv4_shared,
    ) -> c_int;
    pub fn bp_kv4_summarise(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, pool: *const bp_kv4_pool, summary: *const bp_block_summary, pages: *const c_void,
        n_tok: *const c_void, n: u32,
    ) -> c_int;
    pub fn bp_kv4_select(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, summary: *const bp_block_summary,
        args: *const bp_kv4_choice,
    ) -> c_int;
    pub fn bp_kv4_attention_selected(
        ctx: *mut bp_paged_ctx, stream: *mut c_void, dtype: u32, pool: *const bp_kv4_pool, args: *const bp_kv4_chosen,
    ) -> c_int;
}
