//! Bindings of `include/qmm_block.h`: MXFP4 quantisation and product, q/k norm
//! with multi-axis rotary positions, and the norms before and after a block
//! fused with its gate and residual.  One declaration per header entry;
//! `tests/test_block_abi.py` checks that on every change.

use crate::qmm_status;
use core::ffi::c_void;

/// Element type of an operand.
pub type qmm_elem = i32;
pub const QMM_ELEM_BF16: qmm_elem = 0;
pub const QMM_ELEM_F32: qmm_elem = 1;
pub const QMM_ELEM_F16: qmm_elem = 2;

/// Norms of `qmm_gated_residual_norm`.
pub type qmm_norm = i32;
pub const QMM_NORM_NONE: qmm_norm = 0;
pub const QMM_NORM_RMS: qmm_norm = 1;
pub const QMM_NORM_LAYER: qmm_norm = 2;

/// An MXFP4 matrix: E2M1 codes and E8M0 scales in tensor-core order.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct qmm_mx4 {
    pub codes: *const u8,
    pub scales: *const u8,
    pub rows: i64,
    pub k: i64,
}

/// Arguments of `qmm_mx4_linear`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct qmm_mx4_linear_args {
    pub w: qmm_mx4,
    pub m: i64,
    pub x: *const c_void,
    pub x_row_stride: i64,
    pub x_codes: *const u8,
    pub x_scales: *const u8,
    pub bias: *const u16,
    pub gate: *const u16,
    pub residual: *const u16,
    pub y: *mut u16,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
    pub x_elem: i32,
    pub activation: i32,
}

/// Arguments of `qmm_qk_norm_rotary`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct qmm_rotary_args {
    pub q: *const c_void,
    pub k: *const c_void,
    pub q_out: *mut c_void,
    pub k_out: *mut c_void,
    pub q_weight: *const c_void,
    pub k_weight: *const c_void,
    pub positions: *const c_void,
    pub turns: *const f32,
    pub axis: *const u8,
    pub batch: i64,
    pub tokens: i64,
    pub q_stride: [i64; 3],
    pub k_stride: [i64; 3],
    pub q_out_stride: [i64; 3],
    pub k_out_stride: [i64; 3],
    pub pos_batch_stride: i64,
    pub q_heads: i32,
    pub k_heads: i32,
    pub dim: i32,
    pub pairs: i32,
    pub axes: i32,
    pub adjacent: i32,
    pub pos_kind: i32,
    pub elem: i32,
    pub eps: f32,
}

/// Arguments of `qmm_gated_residual_norm`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct qmm_gated_norm_args {
    pub x: *const c_void,
    pub branch: *const c_void,
    pub x_out: *mut c_void,
    pub n_out: *mut c_void,
    pub n_codes: *mut u8,
    pub n_scales: *mut u8,
    pub post_weight: *const c_void,
    pub pre_weight: *const c_void,
    pub gate: *const c_void,
    pub shift: *const c_void,
    pub scale: *const c_void,
    pub rows: i64,
    pub hidden: i64,
    pub x_stride: i64,
    pub branch_stride: i64,
    pub x_out_stride: i64,
    pub n_out_stride: i64,
    pub gate_stride: i64,
    pub shift_stride: i64,
    pub scale_stride: i64,
    pub groups: i64,
    pub x_elem: i32,
    pub branch_elem: i32,
    pub vec_elem: i32,
    pub post: i32,
    pub pre: i32,
    pub residual_scale: f32,
    pub eps: f32,
}

extern "C" {
    pub fn qmm_mx4_code_bytes(rows: i64, k: i64) -> u64;
    pub fn qmm_mx4_scale_bytes(rows: i64, k: i64) -> u64;
    pub fn qmm_mx4_quantize(
        x: *const c_void, elem: i32, rows: i64, k: i64, row_stride: i64, codes: *mut u8, scales: *mut u8,
        stream: *mut c_void,
    ) -> qmm_status;
    pub fn qmm_mx4_dequantize(w: *const qmm_mx4, dst: *mut c_void, elem: i32, stream: *mut c_void) -> qmm_status;
    pub fn qmm_mx4_tile_scales(
        row_major: *const u8, rows: i64, k: i64, scales: *mut u8, stream: *mut c_void,
    ) -> qmm_status;
    pub fn qmm_mx4_row_scales(
        scales: *const u8, rows: i64, k: i64, row_major: *mut u8, stream: *mut c_void,
    ) -> qmm_status;
    pub fn qmm_mx4_workspace_bytes(m: i64, k: i64) -> u64;
    pub fn qmm_mx4_linear_workspace_bytes(m: i64, n: i64, k: i64) -> u64;
    pub fn qmm_mx4_linear(a: *const qmm_mx4_linear_args, stream: *mut c_void) -> qmm_status;
    pub fn qmm_qk_norm_rotary(a: *const qmm_rotary_args, stream: *mut c_void) -> qmm_status;
    pub fn qmm_gated_residual_norm(a: *const qmm_gated_norm_args, stream: *mut c_void) -> qmm_status;
}
