// Bindings of the gfx950 library's 4-bit key/value cache and rotating append
// (include/ullm/kv_cache4.h, include/ullm/kv_rotary.h), for
// crates/ullm-hip-sys.  Written without a Rust toolchain:
// tests/test_kv_rotary_bindings.py checks every constant, struct layout and
// function signature here against the C headers.
//
// Wiring (rust/patches/ullm-hip-sys.patch): `pub mod kv_rotary {
// include!("kv_rotary_bindings.rs"); }` in crates/ullm-hip-sys/src/lib.rs,
// next to the `kv_cache` module.

use core::ffi::c_void;

use crate::kv_cache::{ullm_kv_cache_t, ullm_kv_sequences_t};
use crate::{ullm_error_sink_t, ullm_status_t};

pub const ULLM_KV_CACHE_4_BITS: u32 = 4;
pub const ULLM_KV_ROTARY_INTERLEAVED: u32 = 1;

/// 264 bytes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ullm_kv_cache_append_rotary_desc_t {
    pub struct_size: u32,
    pub abi_version: u32,
    pub cache: *mut ullm_kv_cache_t,
    pub seqs: ullm_kv_sequences_t,
    pub q: *const c_void,
    pub q_row_stride: u64,
    pub q_head_stride: u64,
    pub q_out: *mut c_void,
    pub q_out_row_stride: u64,
    pub q_out_head_stride: u64,
    pub k: *const c_void,
    pub k_row_stride: u64,
    pub k_head_stride: u64,
    pub v: *const c_void,
    pub v_row_stride: u64,
    pub v_head_stride: u64,
    pub weights: *const f32,
    pub inv_freq: *const f32,
    pub positions: *const i32,
    pub position_stride: u64,
    pub pair_axes: *const u8,
    pub heads: u32,
    pub rotary_dims: u32,
    pub axes: u32,
    pub flags: u32,
    pub stream: *mut c_void,
    pub reserved: [u64; 4],
}

unsafe extern "C" {
    pub fn ullm_kv_cache_append_rotary(
        desc: *const ullm_kv_cache_append_rotary_desc_t,
        error_sink: *mut ullm_error_sink_t,
    ) -> ullm_status_t;
}
