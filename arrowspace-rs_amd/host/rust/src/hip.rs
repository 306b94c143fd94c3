// hip.rs -- bindings to include/arrowspace_hip.h (link: -larrowspace_hip).  GENERATED by scripts/gen_rust_bindings.py
// from the header: every export, nothing else.  NOT COMPILED in the build image (no rustc there); the same ABI is
// exercised from C++ (host/arrowspace.hpp, tests/cpp/test_host_mirror.cpp) and from Python (arrowspace_amd/_lib.py).
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_int, c_void};

/// include/arrowspace_hip.h: AS_ABI_VERSION.  The ONE place the Rust side reads the expected version from
/// (shim.rs compares as_abi_version() with it; tests/test_abi.py fails on a literal anywhere else).
pub const AS_ABI_VERSION: c_int = 5;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct AsGraphParams {
    // mirrors GraphParams, src/graph.rs:94-102, plus the two CosinePair variant flags of SURVEY.md Appendix A
    pub eps: f64,
    pub k: u64,
    pub topk: u64,
    pub p: f64,
    pub sigma: f64,
    pub has_sigma: i32,
    pub normalise: i32,
    pub sparsity_check: i32,
    pub rectify: i32,
    pub self_in_results: i32,
    pub reserved: i32,
}
#[repr(C)]
#[derive(Clone, Copy)]
pub struct AsCommOps {
    // the caller's transport for the sharded build: three primitives over device buffers (see the header)
    pub user: *mut c_void,
    pub all_gather_v: Option<unsafe extern "C" fn(*mut c_void, *const c_void, u64, *mut c_void, *const u64, *const u64, *mut c_void) -> c_int>,
    pub all_to_all_v: Option<unsafe extern "C" fn(*mut c_void, *const c_void, *const u64, *const u64, *mut c_void, *const u64, *const u64, *mut c_void) -> c_int>,
    pub all_reduce_sum_u64: Option<unsafe extern "C" fn(*mut c_void, *mut u64, u64, *mut c_void) -> c_int>,
}
#[repr(C)]
pub struct AsCtx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct AsCsr {
    _private: [u8; 0],
}
#[repr(C)]
pub struct AsIndex {
    _private: [u8; 0],
}
#[repr(C)]
pub struct AsJl {
    _private: [u8; 0],
}
#[repr(C)]
pub struct AsComm {
    _private: [u8; 0],
}
#[repr(C)]
pub struct AsTable4 {
    _private: [u8; 0],
}

#[link(name = "arrowspace_hip")]
extern "C" {
    pub fn as_abi_version() -> c_int;
    pub fn as_ctx_create(device: c_int, out: *mut *mut AsCtx) -> c_int;
    pub fn as_ctx_destroy(ctx: *mut AsCtx);
    pub fn as_last_error(ctx: *const AsCtx) -> *const c_char;
    pub fn as_status_message(status: c_int) -> *const c_char;
    pub fn as_ctx_set_stream(ctx: *mut AsCtx, hip_stream: *mut c_void) -> c_int;
    pub fn as_ctx_synchronize(ctx: *mut AsCtx) -> c_int;
    pub fn as_ctx_set_option(ctx: *mut AsCtx, name: *const c_char, value: i64) -> c_int;
    pub fn as_ctx_get_stat(ctx: *const AsCtx, name: *const c_char) -> i64;
    pub fn as_profile_enable(ctx: *mut AsCtx, on: c_int) -> c_int;
    pub fn as_profile_reset(ctx: *mut AsCtx) -> c_int;
    pub fn as_profile_get(ctx: *mut AsCtx, name: *const c_char, ms_total: *mut f64, launches: *mut u64) -> c_int;
    pub fn as_profile_names(ctx: *mut AsCtx, buf: *mut c_char, cap: u64) -> c_int;
    pub fn as_device_upload(ctx: *mut AsCtx, host: *const c_void, bytes: u64, dev_out: *mut *mut c_void) -> c_int;
    pub fn as_device_download(ctx: *mut AsCtx, dev: *const c_void, bytes: u64, host_out: *mut c_void) -> c_int;
    pub fn as_device_free(ctx: *mut AsCtx, dev: *mut c_void);
    pub fn as_define_result_k(k: u64, topk: u64) -> u64;
    pub fn as_build_laplacian(ctx: *mut AsCtx, rows: *const f64, n_nodes: u64, dim: u64, params: *const AsGraphParams, out: *mut *mut AsCsr) -> c_int;
    pub fn as_knn_cosine(ctx: *mut AsCtx, rows: *const f64, n_nodes: u64, dim: u64, row_begin: u64, row_count: u64, params: *const AsGraphParams, nbr_idx: *mut u64, nbr_dist: *mut f64) -> c_int;
    pub fn as_nearest_centroids(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, dim: u64, centroids: *const f64, n_centroids: u64, out_idx: *mut u64, out_dist2: *mut f64) -> c_int;
    pub fn as_two_nn_ratios(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, n_features: u64, sample_ids: *const u64, n_samples: u64, ratios_out: *mut f64) -> c_int;
    pub fn as_kmeans_lloyd(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, n_features: u64, k: u64, max_iter: u64, seed: u64, assignments_out: *mut u64, centroids_out: *mut f64) -> c_int;
    pub fn as_calinski_harabasz(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, n_features: u64, assignments: *const u64, k: u64, score_out: *mut f64) -> c_int;
    pub fn as_compute_optimal_k(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, n_features: u64, seed: u64, k_out: *mut u64, radius_out: *mut f64, id_out: *mut u64) -> c_int;
    pub fn as_incremental_clustering(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, n_features: u64, max_clusters: u64, radius: f64, batch: u64, centroids_out: *mut f64, n_clusters_out: *mut u64, assignments_out: *mut i64, counts_out: *mut u64) -> c_int;
    pub fn as_jl_dimension(n_points: u64, epsilon: f64) -> u64;
    pub fn as_jl_create(ctx: *mut AsCtx, original_dim: u64, reduced_dim: u64, seed: u64, out: *mut *mut AsJl) -> c_int;
    pub fn as_jl_destroy(jl: *mut AsJl);
    pub fn as_jl_original_dim(jl: *const AsJl) -> u64;
    pub fn as_jl_reduced_dim(jl: *const AsJl) -> u64;
    pub fn as_jl_matrix(ctx: *mut AsCtx, jl: *const AsJl, g_out: *mut f64) -> c_int;
    pub fn as_jl_project(ctx: *mut AsCtx, jl: *const AsJl, rows: *const f64, n_rows: u64, out: *mut f64) -> c_int;
    pub fn as_knn_join_applies(ctx: *mut AsCtx, n_nodes: u64, dim: u64, params: *const AsGraphParams) -> c_int;
    pub fn as_knn_join_thresholds(ctx: *mut AsCtx, rows: *const f64, n_nodes: u64, dim: u64, row_begin: u64, row_count: u64, params: *const AsGraphParams, theta_out: *mut f32) -> c_int;
    pub fn as_knn_join_capacity(ctx: *mut AsCtx, params: *const AsGraphParams) -> u32;
    pub fn as_knn_join_pairs(ctx: *mut AsCtx, rows: *const f64, n_nodes: u64, dim: u64, row_begin: u64, row_count: u64, params: *const AsGraphParams, theta_all: *const f32, cap: u32, cnt: *mut u32, cand: *mut u32) -> c_int;
    pub fn as_knn_join_pack(ctx: *mut AsCtx, cnt: *const u32, cand: *const u32, n_rows: u64, cap: u32, row_offsets: *mut u64, packed: *mut u32) -> c_int;
    pub fn as_knn_join_unpack(ctx: *mut AsCtx, cnt: *const u32, packed: *const u32, n_rows: u64, cap: u32, cand_out: *mut u32) -> c_int;
    pub fn as_knn_join_finish(ctx: *mut AsCtx, rows: *const f64, n_nodes: u64, dim: u64, row_begin: u64, row_count: u64, params: *const AsGraphParams, theta_all: *const f32, n_src: u32, cap: u32, cnt_src: *const u32, cand_src: *const u32, nbr_idx: *mut u64, nbr_dist: *mut f64) -> c_int;
    pub fn as_laplacian_from_knn(ctx: *mut AsCtx, nbr_idx: *const u64, nbr_dist: *const f64, n_nodes: u64, params: *const AsGraphParams, out: *mut *mut AsCsr) -> c_int;
    pub fn as_laplacian_from_knn_rows(ctx: *mut AsCtx, nbr_idx: *const u64, nbr_dist: *const f64, n_nodes: u64, params: *const AsGraphParams, row_begin: u64, row_count: u64, out: *mut *mut AsCsr) -> c_int;
    pub fn as_csr_n(m: *const AsCsr) -> u64;
    pub fn as_csr_cols(m: *const AsCsr) -> u64;
    pub fn as_csr_row_begin(m: *const AsCsr) -> u64;
    pub fn as_csr_nnz(m: *const AsCsr) -> u64;
    pub fn as_csr_export(ctx: *mut AsCtx, m: *const AsCsr, indptr: *mut u64, indices: *mut u64, data: *mut f64) -> c_int;
    pub fn as_csr_import(ctx: *mut AsCtx, n: u64, nnz: u64, indptr: *const u64, indices: *const u64, data: *const f64, out: *mut *mut AsCsr) -> c_int;
    pub fn as_csr_free(m: *mut AsCsr);
    pub fn as_comm_unique_id(id128: *mut c_void) -> c_int;
    pub fn as_comm_create_rccl(ctx: *mut AsCtx, id128: *const c_void, rank: c_int, world: c_int, out: *mut *mut AsComm) -> c_int;
    pub fn as_comm_create_custom(ctx: *mut AsCtx, ops: *const AsCommOps, rank: c_int, world: c_int, out: *mut *mut AsComm) -> c_int;
    pub fn as_comm_destroy(comm: *mut AsComm);
    pub fn as_comm_rank(comm: *const AsComm) -> c_int;
    pub fn as_comm_world(comm: *const AsComm) -> c_int;
    pub fn as_shard_range(n: u64, rank: c_int, world: c_int, lo: *mut u64, hi: *mut u64);
    pub fn as_build_laplacian_sharded(ctx: *mut AsCtx, comm: *mut AsComm, rows_shard: *const f64, n_total: u64, dim: u64, params: *const AsGraphParams, out_block: *mut *mut AsCsr, nnz_total: *mut u64) -> c_int;
    pub fn as_lambda_stats_sharded(ctx: *mut AsCtx, comm: *mut AsComm, lambdas_shard: *const f64, n_here: u64, min_out: *mut f64, max_out: *mut f64, mean_out: *mut f64) -> c_int;
    pub fn as_search_lambda_aware_sharded(ctx: *mut AsCtx, comm: *mut AsComm, index_shard: *const AsIndex, queries: *const f64, q_lambdas: *const f64, nq: u64, k: u64, alpha: f64, id_offset: u64, idx_out: *mut u64, score_out: *mut f64) -> c_int;
    pub fn as_compute_taumode_signals_sharded(ctx: *mut AsCtx, comm: *mut AsComm, items_shard: *const f64, n_total: u64, n_features: u64, L_block: *const AsCsr, tau_mode: c_int, tau_arg: f64, lambdas_out: *mut f64) -> c_int;
    pub fn as_compute_taumode(ctx: *mut AsCtx, items: *const f64, n_items: u64, n_features: u64, L: *const AsCsr, tau_mode: c_int, tau_arg: f64, lambdas_out: *mut f64) -> c_int;
    pub fn as_compute_taumode_signals(ctx: *mut AsCtx, items: *const f64, n_items: u64, n_features: u64, L: *const AsCsr, tau_mode: c_int, tau_arg: f64, lambdas_out: *mut f64) -> c_int;
    pub fn as_csr_set_order(ctx: *mut AsCtx, m: *mut AsCsr, order: *const u32) -> c_int;
    pub fn as_prepare_query_items(ctx: *mut AsCtx, queries: *const f64, nq: u64, n_features: u64, L: *const AsCsr, tau_mode: c_int, tau_arg: f64, lambdas_out: *mut f64) -> c_int;
    pub fn as_select_tau(ctx: *mut AsCtx, rows: *const f64, n_rows: u64, len: u64, tau_mode: c_int, tau_arg: f64, taus_out: *mut f64) -> c_int;
    pub fn as_index_create(ctx: *mut AsCtx, items: *const f64, lambdas: *const f64, n_items: u64, n_features: u64, out: *mut *mut AsIndex) -> c_int;
    pub fn as_index_destroy(index: *mut AsIndex);
    pub fn as_index_nitems(index: *const AsIndex) -> u64;
    pub fn as_search_lambda_aware(ctx: *mut AsCtx, index: *const AsIndex, queries: *const f64, q_lambdas: *const f64, nq: u64, k: u64, alpha: f64, id_offset: u64, idx_out: *mut u64, score_out: *mut f64) -> c_int;
    pub fn as_search_lambda_aware_hybrid(ctx: *mut AsCtx, index: *const AsIndex, queries: *const f64, q_lambdas: *const f64, nq: u64, k: u64, alpha: f64, id_offset: u64, idx_out: *mut u64, score_out: *mut f64) -> c_int;
    pub fn as_range_search(ctx: *mut AsCtx, index: *const AsIndex, lambda_q: f64, eps: f64, id_offset: u64, idx_out: *mut u64, dist_out: *mut f64, cap: u64, n_found: *mut u64) -> c_int;
    pub fn as_cross_entropy_workspace(n: u64, n_items: u64, dim: u64, dtype: c_int, backward: c_int) -> u64;
    pub fn as_cross_entropy(ctx: *mut AsCtx, x: *const c_void, n: u64, x_stride: u64, table: *const c_void, n_items: u64, table_stride: u64, dim: u64, dtype: c_int, bias: *const f32, targets: *const i64, ignore_index: i64, scale: f64, losses: *mut f32, lse: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn as_cross_entropy_backward(ctx: *mut AsCtx, x: *const c_void, n: u64, x_stride: u64, table: *const c_void, n_items: u64, table_stride: u64, dim: u64, dtype: c_int, bias: *const f32, targets: *const i64, ignore_index: i64, scale: f64, lse: *const f32, grad_losses: *const f32, grad_lse: *const f32, grad_x: *mut c_void, grad_x_stride: u64, grad_table: *mut c_void, grad_table_stride: u64, grad_bias: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn as_table4_import(ctx: *mut AsCtx, codes: *const u8, scales: *const c_void, zeros: *const u8, n_items: u64, dim: u64, group: u64, scale_dtype: c_int, out: *mut *mut AsTable4) -> c_int;
    pub fn as_table4_pack(ctx: *mut AsCtx, rows: *const c_void, n_items: u64, row_stride: u64, dim: u64, dtype: c_int, group: u64, scale_dtype: c_int, out: *mut *mut AsTable4) -> c_int;
    pub fn as_table4_export(ctx: *mut AsCtx, t: *const AsTable4, codes: *mut u8, scales: *mut c_void, zeros: *mut u8) -> c_int;
    pub fn as_table4_destroy(t: *mut AsTable4);
    pub fn as_table4_items(t: *const AsTable4) -> u64;
    pub fn as_table4_dim(t: *const AsTable4) -> u64;
    pub fn as_table4_group(t: *const AsTable4) -> u64;
    pub fn as_table4_scale_dtype(t: *const AsTable4) -> c_int;
    pub fn as_table4_workspace(t: *const AsTable4, m: u64, dtype: c_int) -> u64;
    pub fn as_table4_scores(ctx: *mut AsCtx, t: *const AsTable4, x: *const c_void, m: u64, x_stride: u64, dtype: c_int, out: *mut c_void, out_stride: u64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
}
