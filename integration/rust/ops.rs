//! The operators of `include/nabla_ops.h` -- embedding lookup, its gradient, dropout -- for a Rust host.
//!
//! UNVERIFIED SOURCE: written against the header by hand; the image this was written in has no
//! Rust toolchain.  `tests/test_ops_cpu.py` checks every declaration below against the header
//! (symbol names, kind and width of each argument, struct fields, constants).
#![allow(dead_code)]

use std::os::raw::{c_int, c_void};

#[repr(C)] pub struct NboMatrix { pub data: *mut c_void, pub rows: u64, pub cols: u64, pub stride: u64,
    pub dtype: i32, pub reserved: i32 }
#[repr(C)] pub struct NboIds { pub data: *const c_void, pub n: u64, pub type_: i32, pub reserved: i32 }
pub enum NboEmbeddingWs {} pub enum NboRng {}

pub const NBO_ID_I32: i32 = 0; pub const NBO_ID_I64: i32 = 1;

#[link(name = "nabla_optim")]
extern "C" {
    pub fn nbo_embedding(table: *const NboMatrix, ids: *const NboIds, add: *const NboMatrix, scale: f64,
                         out: *const NboMatrix) -> c_int;
    pub fn nbo_embedding_ws_create(max_ids: u64, max_cols: u64, out: *mut *mut NboEmbeddingWs) -> c_int;
    pub fn nbo_embedding_ws_destroy(ws: *mut NboEmbeddingWs) -> c_int;
    pub fn nbo_embedding_grad(grad_out: *const NboMatrix, ids: *const NboIds, scale: f64, accumulate: c_int,
                              grad: *const NboMatrix, ws: *mut NboEmbeddingWs) -> c_int;
    pub fn nbo_rng_create(seed: u64, step: u64, out: *mut *mut NboRng) -> c_int;
    pub fn nbo_rng_destroy(rng: *mut NboRng) -> c_int;
    pub fn nbo_rng_state_get(rng: *mut NboRng, seed: *mut u64, step: *mut u64) -> c_int;
    pub fn nbo_rng_load_state(rng: *mut NboRng, seed: u64, step: u64) -> c_int;
    pub fn nbo_rng_advance(rng: *mut NboRng, steps: u64) -> c_int;
    pub fn nbo_dropout(x: *const NboMatrix, residual: *const NboMatrix, p: f64, rng: *mut NboRng, site: u32,
                       out: *const NboMatrix) -> c_int;
}
