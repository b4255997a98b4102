// Bindings of the gfx950 library's key/value cache ABI
// (include/ullm/kv_cache.h), for crates/ullm-hip-sys.  Written without a Rust
// toolchain: tests/test_kv_cache_bindings.py checks every constant, struct
// layout and function signature here against the C header.
//
// Wiring (rust/patches/ullm-hip-sys.patch): `pub mod kv_cache {
// include!("kv_cache_bindings.rs"); }` in crates/ullm-hip-sys/src/lib.rs,
// next to the `linear` module.

use core::ffi::c_void;

use crate::{ullm_error_sink_t, ullm_status_t};

pub const ULLM_KV_CACHE_TRACK_WEIGHTS: u32 = 1;
pub const ULLM_KV_ATTEND_ACCUMULATE: u32 = 1;
pub const ULLM_KV_KERNEL_FEW_ROWS: u32 = 1;
pub const ULLM_KV_KERNEL_MANY_ROWS: u32 = 2;

#[repr(C)]
pub struct ullm_kv_cache_t {
    _private: [u8; 0],
}

/// 72 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub blocks: u64,
    pub block_tokens: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
    pub flags: u32,
    pub device: i32,
    pub reserved0: u32,
    pub reserved: [u64; 4],
}

/// 72 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_info_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub blocks: u64,
    pub block_tokens: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
    pub flags: u32,
    pub device: i32,
    pub reserved0: u32,
    pub device_bytes: u64,
    pub reserved: [u64; 3],
}

/// 56 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_sequences_t {
    pub batch: u64,
    pub rows: u64,
    pub tables: *const i32,
    pub table_stride: u64,
    pub max_blocks: u64,
    pub lengths: *const i32,
    pub starts: *const i32,
}

/// 168 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_append_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub cache: *mut ullm_kv_cache_t,
    pub seqs: ullm_kv_sequences_t,
    pub k: *const c_void,
    pub k_row_stride: u64,
    pub k_head_stride: u64,
    pub v: *const c_void,
    pub v_row_stride: u64,
    pub v_head_stride: u64,
    pub weights: *const f32,
    pub stream: *mut c_void,
    pub reserved: [u64; 4],
}

/// 136 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_gather_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub cache: *const ullm_kv_cache_t,
    pub seqs: ullm_kv_sequences_t,
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub weights: *mut f32,
    pub stream: *mut c_void,
    pub reserved: [u64; 4],
}

/// 200 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_attend_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub cache: *mut ullm_kv_cache_t,
    pub seqs: ullm_kv_sequences_t,
    pub q: *const c_void,
    pub q_row_stride: u64,
    pub q_head_stride: u64,
    pub out: *mut c_void,
    pub out_row_stride: u64,
    pub out_head_stride: u64,
    pub lse: *mut f32,
    pub heads: u32,
    pub window: u32,
    pub scale: f32,
    pub flags: u32,
    pub stream: *mut c_void,
    pub workspace: *mut c_void,
    pub workspace_size: u64,
    pub reserved: [u64; 4],
}

/// 56 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_attend_plan_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub kernel: u32,
    pub row_tile: u32,
    pub parts: u32,
    pub part_tokens: u32,
    pub grid: u64,
    pub workspace_bytes: u64,
    pub reserved: [u64; 2],
}

/// 168 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_evict_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub cache: *mut ullm_kv_cache_t,
    pub seqs: ullm_kv_sequences_t,
    pub new_tables: *const i32,
    pub new_table_stride: u64,
    pub new_lengths: *mut i32,
    pub kept: *mut i32,
    pub keep: u64,
    pub sink: u64,
    pub recent: u64,
    pub stream: *mut c_void,
    pub reserved: [u64; 4],
}

unsafe extern "C" {
    pub fn ullm_kv_cache_create(
        desc: *const ullm_kv_cache_desc_t,
        cache: *mut *mut ullm_kv_cache_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_destroy(
        cache: *mut *mut ullm_kv_cache_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_query(
        cache: *const ullm_kv_cache_t,
        info: *mut ullm_kv_cache_info_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_append(
        desc: *const ullm_kv_cache_append_desc_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_gather(
        desc: *const ullm_kv_cache_gather_desc_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_attend(
        desc: *const ullm_kv_cache_attend_desc_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_attend_plan(
        desc: *const ullm_kv_cache_attend_desc_t,
        plan: *mut ullm_kv_attend_plan_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
    pub fn ullm_kv_cache_evict(
        desc: *const ullm_kv_cache_evict_desc_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
}
