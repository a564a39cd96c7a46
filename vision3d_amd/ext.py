"""Drop-in for the CUDA half of the reference's ``vision3d.ext`` pybind11 module.

Same function names, positional order and keyword names as ``/root/reference/vision3d/csrc/pybind.cpp:71-158``;
same contract: the caller pre-allocates every output tensor, the call writes in place, returns ``None``, runs
asynchronously on the current stream of the tensors' device and validates its arguments with the reference's
messages (``csrc/common/torch_helper.h:9-23``).  Underneath, each call is one C-ABI call into
``libv3d_hip.so`` (``include/v3d_hip.h``) -- hand-written gfx950 kernels, no fallback.

``knn`` is an alias of ``knn_points``: the reference's Python wrapper calls ``ext_module.knn``
(``ops/knn_points.py:36``) although the extension registers ``knn_points`` (``pybind.cpp:150``).
"""
import ctypes

import torch

from . import _lib

__all__ = [
    "ball_query",
    "ball_query_multi",
    "furthest_point_sample",
    "furthest_point_sample_rounds",
    "gather_forward",
    "gather_backward",
    "group_gather_forward",
    "group_gather_backward",
    "three_nn",
    "three_interpolate_forward",
    "three_interpolate_backward",
    "knn_points",
    "knn",
    "pairwise_distance",
    "radius_count",
    "radius_count_pack",
    "knn_feat",
    "topk_merge",
    "radius_search_pack",
    "grid_subsample_pack",
    "voxelize_pack",
    "mutual_topk_select",
    "mutual_select_lists",
    "threshold_select",
    "global_topk_select",
    "index_select_rows",
    "local_maxpool_pack",
    "knn_interp_weights_pack",
    "rows_weighted_sum",
    "global_avgpool_pack",
    "rows_csr_build",
    "rows_scatter",
    "sa_group",
    "edge_group",
    "kpconv_gather",
    "kpconv_gather_backward",
    "point_to_node_partition",
    "point_to_node_knn",
    "attention_pack_forward",
    "attention_pack_backward",
    "cached_attention",
    "layer_norm_forward",
    "layer_norm_backward",
    "radius_neighbors",
    "grid_subsampling",
    "sample_nodes_with_fps",
]

_FLOATING = {torch.float32: "f32", torch.float64: "f64"}
# AT_DISPATCH_ALL_TYPES_AND(Bool) of gather_cuda.cu:22 / group_gather_cuda.cu:23
_ALL_AND_BOOL = {
    torch.uint8: 1, torch.int8: 1, torch.bool: 1, torch.int16: 2, torch.int32: 4, torch.float32: 4,
    torch.int64: 8, torch.float64: 8,
}
_TYPE_NAMES = {torch.float16: "Half", torch.bfloat16: "BFloat16", torch.float32: "Float", torch.float64: "Double",
               torch.int32: "Int", torch.int64: "Long", torch.int16: "Short", torch.int8: "Char",
               torch.uint8: "Byte", torch.bool: "Bool"}


def _check_cuda_contiguous(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _check_long(t, name):
    if t.dtype != torch.int64:
        raise RuntimeError(f"{name} must be an long tensor")


def _check_float(t, name):
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} must be a float tensor")


def _floating_suffix(t, kernel):
    try:
        return _FLOATING[t.dtype]
    except KeyError:
        raise RuntimeError(f'"{kernel}" not implemented for \'{_TYPE_NAMES.get(t.dtype, t.dtype)}\'') from None


def _same_dtype(kernel, ref, *others):
    for o in others:
        if o.dtype != ref.dtype:
            raise RuntimeError(f"{kernel}: expected scalar type {_TYPE_NAMES.get(ref.dtype, ref.dtype)} but found "
                               f"{_TYPE_NAMES.get(o.dtype, o.dtype)}")


def _where(t):
    """(device index, raw hipStream_t) of the current stream on the tensor's device."""
    dev = t.get_device()
    return dev, torch._C._cuda_getCurrentRawStream(dev)  # current_stream(dev).cuda_stream without the Stream object


def _workspace(nbytes, like):
    """Scratch from torch's caching allocator (stream-ordered reuse, no hipMalloc on the hot path)."""
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=like.device)


def _ws_args(nbytes, like):
    """(tensor kept alive by the caller, pointer, size) of a torch-owned workspace; a call that needs no scratch gets
    (None, NULL, 0).  torch's allocations are 512-byte aligned, which covers the ABI's 256."""
    nbytes = int(nbytes)
    if nbytes == 0:
        return None, None, 0
    ws = _workspace(nbytes, like)
    return ws, ws.data_ptr(), ws.numel()


# --------------------------------------------------------------------------------------------------------
def ball_query_multi(q_points, s_points, indices_list, max_radii, num_samples_list):
    """Multi-scale ball query (PointNet++ MSG): up to four (radius, k) scales over the same clouds in one pass; every
    ``indices_list[i]`` (B, M, num_samples_list[i]) arrives zero-filled and leaves equal to ``ball_query`` of that scale."""
    n = len(indices_list)
    if not (1 <= n <= 4) or len(max_radii) != n or len(num_samples_list) != n:
        raise RuntimeError("ball_query_multi: 1 to 4 scales, one radius and one sample count per output")
    _check_cuda_contiguous(q_points, "q_points")
    _check_cuda_contiguous(s_points, "s_points")
    _check_float(q_points, "q_points")
    _check_float(s_points, "s_points")
    B, M, N = q_points.size(0), q_points.size(1), s_points.size(1)
    for t, k in zip(indices_list, num_samples_list):
        _check_cuda_contiguous(t, "indices")
        _check_long(t, "indices")
        if tuple(t.shape) != (B, M, int(k)):
            raise RuntimeError(f"ball_query_multi: indices must have shape {(B, M, int(k))}")
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in indices_list])
    radii = (ctypes.c_float * n)(*[float(r) for r in max_radii])
    ks = (ctypes.c_int * n)(*[int(k) for k in num_samples_list])
    dev, stream = _where(q_points)
    _lib.check(_lib.lib().v3d_ball_query_multi_f32(q_points.data_ptr(), s_points.data_ptr(), ptrs, radii, ks, n, B, M, N,
                                                   dev, stream), "ball_query_multi")


def ball_query(q_points, s_points, indices, max_radius, num_samples):
    _check_cuda_contiguous(q_points, "q_points")
    _check_cuda_contiguous(s_points, "s_points")
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    sfx = _floating_suffix(q_points, "ball_query_kernel")
    _same_dtype("ball_query", q_points, s_points)
    B, M, N = q_points.size(0), q_points.size(1), s_points.size(1)
    dev, stream = _where(q_points)
    fn = getattr(_lib.lib(), "v3d_ball_query_" + sfx)
    _lib.check(fn(q_points.data_ptr(), s_points.data_ptr(), indices.data_ptr(), B, M, N, float(max_radius),
                  int(num_samples), dev, stream), "ball_query")


def furthest_point_sample(points, distances, indices, num_samples):
    furthest_point_sample_rounds(points, distances, indices, num_samples, 0, num_samples)


def furthest_point_sample_rounds(points, distances, indices, num_samples, first, last):
    """Not in the reference's extension: only the rounds [first, last) of the sampling of ``num_samples`` points, the
    rounds before them already in ``indices[:, :first]`` and the running distances in ``distances`` (first % 64 == 0).
    For callers that start the consumers of the first samples while the sampling goes on (v3d_fps_resume_f32)."""
    _check_cuda_contiguous(points, "points")
    _check_cuda_contiguous(distances, "distances")
    _check_cuda_contiguous(indices, "indices")
    _check_float(points, "points")
    _check_float(distances, "distances")
    _check_long(indices, "indices")
    B, N = points.size(0), points.size(1)
    dev, stream = _where(points)
    _lib.check(_lib.lib().v3d_fps_resume_f32(points.data_ptr(), distances.data_ptr(), indices.data_ptr(), B, N,
                                             int(num_samples), int(first), int(last), dev, stream),
               "furthest_point_sample")


def _gather_forward(name, kernel, sources, indices, targets, grouped):
    _check_cuda_contiguous(sources, "sources")
    _check_cuda_contiguous(indices, "indices")
    _check_cuda_contiguous(targets, "targets")
    _check_long(indices, "indices")
    try:
        elem = _ALL_AND_BOOL[sources.dtype]
    except KeyError:
        raise RuntimeError(f'"{kernel}" not implemented for \'{_TYPE_NAMES.get(sources.dtype, sources.dtype)}\'') from None
    _same_dtype(name, sources, targets)
    B, C, N = sources.size(0), sources.size(1), sources.size(2)
    dev, stream = _where(sources)
    if grouped:
        rc = _lib.lib().v3d_group_gather_fwd(sources.data_ptr(), indices.data_ptr(), targets.data_ptr(), B, C, N,
                                             indices.size(1), indices.size(2), elem, dev, stream)
    else:
        rc = _lib.lib().v3d_gather_fwd(sources.data_ptr(), indices.data_ptr(), targets.data_ptr(), B, C, N,
                                       indices.size(1), elem, dev, stream)
    _lib.check(rc, name)


def gather_forward(sources, indices, targets):
    _gather_forward("gather_forward", "gather_forward_kernel", sources, indices, targets, grouped=False)


def group_gather_forward(sources, indices, targets):
    _gather_forward("group_gather_forward", "group_gather_forward_kernel", sources, indices, targets, grouped=True)


class ScatterLists:
    """The inversion of one index tensor (v3d_scatter_build): the device workspace that holds the lists and what they were
    built for.  Kept by the caller (the ops cache it on the index tensor) and handed to every backward that flows through
    those indices."""
    __slots__ = ("workspace", "mode", "B", "N", "L", "weights")

    def __init__(self, workspace, mode, B, N, L, weights):
        self.workspace, self.mode, self.B, self.N, self.L, self.weights = workspace, mode, B, N, L, weights


def scatter_build(indices, num_sources, weights=None):
    """Not in the reference's extension (its backward kernels scatter with atomics): inverts ``indices`` -- (B, M) /
    (B, M, K) of gather / group_gather, or the (B, Q, 3) table of three_interpolate together with its ``weights`` -- into
    per-source lists once; ``scatter_apply`` then only sums, as often as wanted."""
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    mode, elem = 0, 4
    if weights is not None:
        _check_cuda_contiguous(weights, "weights")
        _floating_suffix(weights, "three_interpolate_backward_kernel")
        if tuple(weights.shape) != tuple(indices.shape) or indices.dim() != 3 or indices.size(2) != 3:
            raise RuntimeError("scatter_build: three_interpolate lists need indices and weights of shape (B, Q, 3)")
        mode, elem = 1, weights.element_size()
    B, N = indices.size(0), int(num_sources)
    L = indices.numel() // max(B, 1)
    dev, stream = _where(indices)
    nbytes = _lib.lib().v3d_scatter_workspace_bytes(B, N, L)
    ws = torch.empty((max(nbytes, 256) + 256,), dtype=torch.uint8, device=indices.device)
    ws = ws[(-ws.data_ptr()) % 256:][:max(nbytes, 256)]  # 256-byte aligned, owned by the lists (not the shared scratch)
    rc = _lib.lib().v3d_scatter_build(indices.data_ptr(), 0 if weights is None else weights.data_ptr(), mode, elem, B, N, L,
                                      ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "scatter_build")
    return ScatterLists(ws, mode, B, N, L, weights)


def _scatter_apply(name, target_grads, lists, source_grads, sfx, L, mode):
    B, C = target_grads.size(0), target_grads.size(1)
    if (lists.mode, lists.B, lists.L, lists.N) != (mode, B, L, source_grads.size(2)):
        raise RuntimeError(f"{name}: the lists were built for another index tensor (mode / B / positions / sources differ)")
    dev, stream = _where(target_grads)
    fn = getattr(_lib.lib(), "v3d_scatter_apply_" + sfx)
    w = 0 if lists.weights is None else lists.weights.data_ptr()
    _lib.check(fn(target_grads.data_ptr(), w, source_grads.data_ptr(), mode, B, C, lists.N, L, lists.workspace.data_ptr(),
                  lists.workspace.numel(), dev, stream), name)


def _gather_backward(name, kernel, target_grads, indices, source_grads, num_sources, grouped):
    _check_cuda_contiguous(target_grads, "target_grads")
    _check_cuda_contiguous(indices, "indices")
    _check_cuda_contiguous(source_grads, "source_grads")
    _check_long(indices, "indices")
    sfx = _floating_suffix(target_grads, kernel)
    _same_dtype(name, target_grads, source_grads)
    B, C = target_grads.size(0), target_grads.size(1)
    N = int(num_sources)
    if source_grads.size(2) != N:
        raise RuntimeError(f"{name}: source_grads has {source_grads.size(2)} sources, num_sources={N}")
    dev, stream = _where(target_grads)
    L = target_grads.size(2) * (target_grads.size(3) if grouped else 1)
    nbytes = _lib.lib().v3d_scatter_workspace_bytes(B, N, L)
    ws = _workspace(nbytes, target_grads)
    if grouped:
        fn = getattr(_lib.lib(), "v3d_group_gather_bwd_" + sfx)
        rc = fn(target_grads.data_ptr(), indices.data_ptr(), source_grads.data_ptr(), B, C, N, target_grads.size(2),
                target_grads.size(3), ws.data_ptr(), ws.numel(), dev, stream)
    else:
        fn = getattr(_lib.lib(), "v3d_gather_bwd_" + sfx)
        rc = fn(target_grads.data_ptr(), indices.data_ptr(), source_grads.data_ptr(), B, C, N, target_grads.size(2),
                ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, name)


def gather_backward(target_grads, indices, source_grads, num_sources):
    _gather_backward("gather_backward", "gather_backward_kernel", target_grads, indices, source_grads, num_sources,
                     grouped=False)


def group_gather_backward(target_grads, indices, source_grads, num_sources):
    _gather_backward("group_gather_backward", "group_gather_backward_kernel", target_grads, indices, source_grads,
                     num_sources, grouped=True)


def scatter_apply(target_grads, lists, source_grads):
    """Not in the reference's extension: the backward of gather / group_gather / three_interpolate with the lists of
    ``scatter_build`` -- ``source_grads`` (B, C, num_sources) fully written from ``target_grads`` (B, C, M) / (B, C, M, K) /
    (B, C, Q), bit-identical to ``gather_backward`` / ``group_gather_backward`` / ``three_interpolate_backward``."""
    _check_cuda_contiguous(target_grads, "target_grads")
    _check_cuda_contiguous(source_grads, "source_grads")
    kernel = "three_interpolate_backward_kernel" if lists.mode == 1 else "group_gather_backward_kernel"
    sfx = _floating_suffix(target_grads, kernel)
    _same_dtype("scatter_apply", target_grads, source_grads)
    if lists.weights is not None:
        _same_dtype("scatter_apply", target_grads, lists.weights)
    positions = target_grads.numel() // max(target_grads.size(0) * target_grads.size(1), 1)
    _scatter_apply("scatter_apply", target_grads, lists, source_grads, sfx, positions * (3 if lists.mode == 1 else 1),
                   lists.mode)


def three_nn(q_points, s_points, tnn_distances, tnn_indices):
    _check_cuda_contiguous(q_points, "q_points")
    _check_cuda_contiguous(s_points, "s_points")
    _check_cuda_contiguous(tnn_distances, "tnn_distances")
    _check_cuda_contiguous(tnn_indices, "tnn_indices")
    _check_long(tnn_indices, "tnn_indices")
    sfx = _floating_suffix(q_points, "three_nn_kernel")
    _same_dtype("three_nn", q_points, s_points, tnn_distances)
    B, Q, S = q_points.size(0), q_points.size(1), s_points.size(1)
    dev, stream = _where(q_points)
    fn = getattr(_lib.lib(), "v3d_three_nn_" + sfx)
    _lib.check(fn(q_points.data_ptr(), s_points.data_ptr(), tnn_distances.data_ptr(), tnn_indices.data_ptr(), B, Q, S,
                  dev, stream), "three_nn")


def three_interpolate_forward(sources, indices, weights, targets):
    _check_cuda_contiguous(sources, "sources")
    _check_cuda_contiguous(indices, "indices")
    _check_cuda_contiguous(weights, "weights")
    _check_cuda_contiguous(targets, "targets")
    _check_long(indices, "indices")
    sfx = _floating_suffix(sources, "three_interpolate_forward_kernel")
    _same_dtype("three_interpolate_forward", sources, weights, targets)
    B, C, S = sources.size(0), sources.size(1), sources.size(2)
    Q = indices.size(1)
    dev, stream = _where(sources)
    fn = getattr(_lib.lib(), "v3d_three_interp_fwd_" + sfx)
    _lib.check(fn(sources.data_ptr(), indices.data_ptr(), weights.data_ptr(), targets.data_ptr(), B, C, S, Q, dev,
                  stream), "three_interpolate_forward")


def three_interpolate_backward(target_grads, indices, weights, source_grads, num_sources):
    _check_cuda_contiguous(target_grads, "target_grads")
    _check_cuda_contiguous(indices, "indices")
    _check_cuda_contiguous(weights, "weights")
    _check_cuda_contiguous(source_grads, "source_grads")
    _check_long(indices, "indices")
    sfx = _floating_suffix(target_grads, "three_interpolate_backward_kernel")
    _same_dtype("three_interpolate_backward", target_grads, weights, source_grads)
    B, C, Q = target_grads.size(0), target_grads.size(1), target_grads.size(2)
    S = int(num_sources)
    if source_grads.size(2) != S:
        raise RuntimeError(f"three_interpolate_backward: source_grads has {source_grads.size(2)} sources, "
                           f"num_sources={S}")
    dev, stream = _where(target_grads)
    nbytes = _lib.lib().v3d_scatter_workspace_bytes(B, S, Q * 3)
    ws = _workspace(nbytes, target_grads)
    fn = getattr(_lib.lib(), "v3d_three_interp_bwd_" + sfx)
    rc = fn(target_grads.data_ptr(), indices.data_ptr(), weights.data_ptr(), source_grads.data_ptr(), B, C, S, Q,
            ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "three_interpolate_backward")


def knn_points(q_points, s_points, knn_distances, knn_indices, num_neighbors):
    _check_cuda_contiguous(q_points, "q_points")
    _check_cuda_contiguous(s_points, "s_points")
    _check_cuda_contiguous(knn_distances, "knn_distances")
    _check_cuda_contiguous(knn_indices, "knn_indices")
    _check_long(knn_indices, "knn_indices")
    sfx = _floating_suffix(q_points, "knn_points_kernel")
    _same_dtype("knn_points", q_points, s_points, knn_distances)
    B, M, N = q_points.size(0), q_points.size(1), s_points.size(1)
    dev, stream = _where(q_points)
    fn = getattr(_lib.lib(), "v3d_knn_points_" + sfx)
    _lib.check(fn(q_points.data_ptr(), s_points.data_ptr(), knn_distances.data_ptr(), knn_indices.data_ptr(), B, M, N,
                  int(num_neighbors), dev, stream), "knn_points")


knn = knn_points  # ops/knn_points.py:36 calls ext_module.knn


# --------------------------------------------------------------------------------------------------------
# Entry points without a counterpart in the reference extension: the reference computes these with
# torch.matmul + elementwise passes (ops/pairwise_distance.py) and with pykeops (ops/knn.py).
# --------------------------------------------------------------------------------------------------------
def pairwise_distance(x, y, out, normalized=False, squared=True, eps=1e-8, strict=False):
    """x (batch,N,C), y (batch,M,C), out (batch,N,M); fp32, contiguous, in place."""
    for t, name in ((x, "x"), (y, "y"), (out, "out")):
        _check_cuda_contiguous(t, name)
        _check_float(t, name)
    batch, N, C = x.shape
    M = y.shape[1]
    flags = (1 if normalized else 0) | (0 if squared else 2) | (4 if strict else 0)
    dev, stream = _where(x)
    _lib.check(_lib.lib().v3d_pairwise_distance_f32(x.data_ptr(), y.data_ptr(), out.data_ptr(), batch, N, M, C, flags,
                                                    float(eps), dev, stream), "pairwise_distance")


def radius_count(q_points, s_points, counts, radius):
    """q (B,M,3), s (B,N,3) fp32 -> counts (B,M) int64 of supports strictly closer than ``radius``."""
    _check_cuda_contiguous(q_points, "q_points")
    _check_cuda_contiguous(s_points, "s_points")
    _check_cuda_contiguous(counts, "counts")
    _check_float(q_points, "q_points")
    _check_float(s_points, "s_points")
    _check_long(counts, "counts")
    B, M, N = q_points.size(0), q_points.size(1), s_points.size(1)
    dev, stream = _where(q_points)
    _lib.check(_lib.lib().v3d_radius_count_f32(q_points.data_ptr(), s_points.data_ptr(), counts.data_ptr(), B, M, N,
                                               float(radius), dev, stream), "radius_count")


def knn_feat(x, y, distances, indices, num_neighbors, index_offset=0):
    """x (batch,N,C), y (batch,M,C) -> distances (batch,N,k) fp32 (Euclidean), indices (batch,N,k) int64."""
    for t, name in ((x, "x"), (y, "y"), (distances, "distances")):
        _check_cuda_contiguous(t, name)
        _check_float(t, name)
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    batch, N, C = x.shape
    M = y.shape[1]
    k = int(num_neighbors)
    dev, stream = _where(x)
    nbytes = _lib.lib().v3d_knn_feat_workspace_bytes(batch, N, max(M, 1), C, k)
    ws = _workspace(nbytes, x)
    rc = _lib.lib().v3d_knn_feat_f32(x.data_ptr(), y.data_ptr(), distances.data_ptr(), indices.data_ptr(), batch, N, M,
                                     C, k, int(index_offset), ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "knn_feat")


def topk_merge(parts_distances, parts_indices, distances, indices):
    """parts (G,rows,k) sorted partial lists -> (rows,k) global top-k by (distance, index)."""
    _check_cuda_contiguous(parts_distances, "parts_distances")
    _check_cuda_contiguous(parts_indices, "parts_indices")
    _check_cuda_contiguous(distances, "distances")
    _check_cuda_contiguous(indices, "indices")
    _check_float(parts_distances, "parts_distances")
    _check_float(distances, "distances")
    _check_long(parts_indices, "parts_indices")
    _check_long(indices, "indices")
    G, rows, k = parts_distances.shape
    dev, stream = _where(parts_distances)
    _lib.check(_lib.lib().v3d_topk_merge_f32(parts_distances.data_ptr(), parts_indices.data_ptr(),
                                             distances.data_ptr(), indices.data_ptr(), G, rows, k, dev, stream),
               "topk_merge")


def radius_search_pack(q_points, s_points, q_lengths, s_lengths, neighbor_indices, radius, neighbor_limit):
    """q_points (M,3), s_points (N,3) fp32; lengths (B,) int64 on the same device; neighbor_indices (M, limit) int64."""
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (q_lengths, "q_lengths"),
                    (s_lengths, "s_lengths"), (neighbor_indices, "neighbor_indices")):
        _check_cuda_contiguous(t, name)
    _check_float(q_points, "q_points")
    _check_float(s_points, "s_points")
    for t, name in ((q_lengths, "q_lengths"), (s_lengths, "s_lengths"), (neighbor_indices, "neighbor_indices")):
        _check_long(t, name)
    B = q_lengths.shape[0]
    if s_lengths.shape[0] != B:
        raise RuntimeError("q_lengths and s_lengths must have the same number of clouds")
    M, N = q_points.shape[0], s_points.shape[0]
    dev, stream = _where(q_points)
    ws = _workspace(_lib.lib().v3d_radius_search_workspace_bytes(B, N), q_points)
    rc = _lib.lib().v3d_radius_search_pack_f32(
        q_points.data_ptr(), s_points.data_ptr(), q_lengths.data_ptr(), s_lengths.data_ptr(),
        neighbor_indices.data_ptr(), B, M, N, float(radius), int(neighbor_limit), ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "radius_search_pack_mode")


class RadiusGrid:
    """The cell list of one support set (``radius_grid_build``): serves ``radius_search_grid`` at every radius up to
    ``cell_radius``.  Searches on one grid must be stream-ordered (each rewrites the query offsets kept in it)."""

    __slots__ = ("workspace", "num_clouds", "num_supports", "cell_radius", "s_points", "s_lengths")

    def __init__(self, workspace, num_clouds, num_supports, cell_radius, s_points, s_lengths):
        self.workspace, self.num_clouds, self.num_supports = workspace, num_clouds, num_supports
        self.cell_radius, self.s_points, self.s_lengths = cell_radius, s_points, s_lengths  # (inputs kept alive)


def radius_grid_build(s_points, s_lengths, cell_radius):
    """s_points (N,3) fp32, s_lengths (B,) int64 on the same device -> RadiusGrid for radii <= cell_radius."""
    _check_cuda_contiguous(s_points, "s_points")
    _check_cuda_contiguous(s_lengths, "s_lengths")
    _check_float(s_points, "s_points")
    _check_long(s_lengths, "s_lengths")
    B, N = s_lengths.shape[0], s_points.shape[0]
    dev, stream = _where(s_points)
    ws = _workspace(_lib.lib().v3d_radius_search_workspace_bytes(B, N), s_points)
    _lib.check(_lib.lib().v3d_radius_grid_build_f32(s_points.data_ptr(), s_lengths.data_ptr(), B, N, float(cell_radius),
                                                   ws.data_ptr(), ws.numel(), dev, stream), "radius_grid_build")
    return RadiusGrid(ws, B, N, float(cell_radius), s_points, s_lengths)


def radius_search_grid(q_points, q_lengths, grid, neighbor_indices, radius, neighbor_limit):
    """``radius_search_pack`` against the supports of ``grid`` (identical result); radius <= grid.cell_radius."""
    for t, name in ((q_points, "q_points"), (q_lengths, "q_lengths"), (neighbor_indices, "neighbor_indices")):
        _check_cuda_contiguous(t, name)
    _check_float(q_points, "q_points")
    _check_long(q_lengths, "q_lengths")
    _check_long(neighbor_indices, "neighbor_indices")
    if q_lengths.shape[0] != grid.num_clouds:
        raise RuntimeError("q_lengths and the grid must have the same number of clouds")
    M = q_points.shape[0]
    if neighbor_indices.numel() != M * int(neighbor_limit):
        raise RuntimeError("neighbor_indices must hold neighbor_limit entries per query")
    dev, stream = _where(q_points)
    _lib.check(_lib.lib().v3d_radius_search_grid_f32(
        q_points.data_ptr(), q_lengths.data_ptr(), neighbor_indices.data_ptr(), grid.num_clouds, M, grid.num_supports,
        grid.cell_radius, float(radius), int(neighbor_limit), grid.workspace.data_ptr(), grid.workspace.numel(), dev,
        stream), "radius_search_grid")


def knn_lex(q_points, s_points, knn_distances, knn_indices, num_neighbors):
    """q_points (B,M,3), s_points (B,N,3) fp32 -> knn_distances (B,M,k) ascending, knn_indices (B,M,k) int64; equal
    distances lower index first (the order pykeops' Kmin_argKmin yields; ``knn_points`` keeps the CUDA heap's)."""
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (knn_distances, "knn_distances"),
                    (knn_indices, "knn_indices")):
        _check_cuda_contiguous(t, name)
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (knn_distances, "knn_distances")):
        _check_float(t, name)
    _check_long(knn_indices, "knn_indices")
    B, M, N, k = q_points.size(0), q_points.size(1), s_points.size(1), int(num_neighbors)
    if q_points.size(-1) != 3 or s_points.size(-1) != 3 or s_points.size(0) != B:
        raise RuntimeError("knn_lex: points must be (B, M, 3) and (B, N, 3)")
    if knn_distances.numel() != B * M * k or knn_indices.numel() != B * M * k:
        raise RuntimeError("knn_lex: distances / indices must hold k entries per query")
    dev, stream = _where(q_points)
    _lib.check(_lib.lib().v3d_knn_lex_f32(q_points.data_ptr(), s_points.data_ptr(), knn_distances.data_ptr(),
                                         knn_indices.data_ptr(), B, M, N, k, dev, stream), "knn")


def knn_pack(q_points, s_points, q_lengths, s_lengths, distances, indices, num_neighbors):
    """q_points (M,3), s_points (N,3) fp32; lengths (B,) int64 on the same device -> distances (M,k) fp32, indices (M,k)
    int64 = positions inside the query's own cloud, equal distances lower index first (pykeops' order).  k <= 100."""
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (q_lengths, "q_lengths"), (s_lengths, "s_lengths"),
                    (distances, "distances"), (indices, "indices")):
        _check_cuda_contiguous(t, name)
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (distances, "distances")):
        _check_float(t, name)
    for t, name in ((q_lengths, "q_lengths"), (s_lengths, "s_lengths"), (indices, "indices")):
        _check_long(t, name)
    B = q_lengths.shape[0]
    if s_lengths.shape[0] != B:
        raise RuntimeError("q_lengths and s_lengths must have the same number of clouds")
    M, N, k = q_points.shape[0], s_points.shape[0], int(num_neighbors)
    if q_points.shape[-1] != 3 or s_points.shape[-1] != 3:
        raise RuntimeError("knn_pack: points must be (N, 3)")
    if distances.numel() != M * k or indices.numel() != M * k:
        raise RuntimeError("knn_pack: distances / indices must hold k entries per query")
    dev, stream = _where(q_points)
    ws = _workspace(_lib.lib().v3d_knn_pack_workspace_bytes(B, N, k), q_points)
    rc = _lib.lib().v3d_knn_pack_f32(
        q_points.data_ptr(), s_points.data_ptr(), q_lengths.data_ptr(), s_lengths.data_ptr(), distances.data_ptr(),
        indices.data_ptr(), B, M, N, k, ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "knn_pack_mode")


def radius_count_pack(q_points, s_points, q_lengths, s_lengths, counts, radius):
    """q_points (M,3), s_points (N,3) fp32; lengths (B,) int64 on the same device; counts (M,) int64."""
    for t, name in ((q_points, "q_points"), (s_points, "s_points"), (q_lengths, "q_lengths"),
                    (s_lengths, "s_lengths"), (counts, "counts")):
        _check_cuda_contiguous(t, name)
    _check_float(q_points, "q_points")
    _check_float(s_points, "s_points")
    for t, name in ((q_lengths, "q_lengths"), (s_lengths, "s_lengths"), (counts, "counts")):
        _check_long(t, name)
    B = q_lengths.shape[0]
    if s_lengths.shape[0] != B:
        raise RuntimeError("q_lengths and s_lengths must have the same number of clouds")
    M, N = q_points.shape[0], s_points.shape[0]
    if counts.numel() != M:
        raise RuntimeError("radius_count_pack: counts must hold one entry per query")
    dev, stream = _where(q_points)
    ws = _workspace(_lib.lib().v3d_radius_search_workspace_bytes(B, N), q_points)
    rc = _lib.lib().v3d_radius_count_pack_f32(
        q_points.data_ptr(), s_points.data_ptr(), q_lengths.data_ptr(), s_lengths.data_ptr(), counts.data_ptr(), B, M, N,
        float(radius), ws.data_ptr(), ws.numel(), dev, stream)
    _lib.check(rc, "radius_count_pack_mode")


def grid_subsample_pack(points, lengths, sampled_points, sampled_lengths, num_sampled, voxel_size):
    """points (N,3) fp32, lengths (B,) int64 -> sampled_points (N,3) capacity, sampled_lengths (B,), num_sampled ()."""
    for t, name in ((points, "points"), (lengths, "lengths"), (sampled_points, "sampled_points"),
                    (sampled_lengths, "sampled_lengths"), (num_sampled, "num_sampled")):
        _check_cuda_contiguous(t, name)
    _check_float(points, "points")
    _check_float(sampled_points, "sampled_points")
    for t, name in ((lengths, "lengths"), (sampled_lengths, "sampled_lengths"), (num_sampled, "num_sampled")):
        _check_long(t, name)
    if sampled_points.shape[0] < points.shape[0] or sampled_lengths.shape[0] != lengths.shape[0]:
        raise RuntimeError("grid_subsample_pack: output buffers too small")
    dev, stream = _where(points)
    ws, wp, wn = _ws_args(_lib.lib().v3d_grid_subsample_workspace_bytes(lengths.shape[0], points.shape[0], 0), points)
    rc = _lib.lib().v3d_grid_subsample_pack_f32(
        points.data_ptr(), lengths.data_ptr(), sampled_points.data_ptr(), sampled_lengths.data_ptr(),
        num_sampled.data_ptr(), lengths.shape[0], points.shape[0], float(voxel_size), wp, wn, dev, stream)
    _lib.check(rc, "grid_subsample_pack_mode")


def voxelize_pack(points, lengths, voxels, nodes, voxel_lengths, num_voxels, voxel_size, feats=None, voxel_feats=None):
    """points (N,3) fp32, lengths (B,), optional feats (N,C) -> voxels (N,3) i64 / nodes (N,3) / voxel_feats (N,C)
    capacity buffers, voxel_lengths (B,), num_voxels ()."""
    for t, name in ((points, "points"), (lengths, "lengths"), (voxels, "voxels"), (nodes, "nodes"),
                    (voxel_lengths, "voxel_lengths"), (num_voxels, "num_voxels")):
        _check_cuda_contiguous(t, name)
    _check_float(points, "points")
    _check_float(nodes, "nodes")
    for t, name in ((lengths, "lengths"), (voxels, "voxels"), (voxel_lengths, "voxel_lengths"),
                    (num_voxels, "num_voxels")):
        _check_long(t, name)
    n = points.shape[0]
    if voxels.shape[0] < n or nodes.shape[0] < n or voxel_lengths.shape[0] != lengths.shape[0]:
        raise RuntimeError("voxelize_pack: output buffers too small")
    C = 0
    if feats is not None:
        _check_cuda_contiguous(feats, "feats")
        _check_float(feats, "feats")
        if voxel_feats is None:
            raise RuntimeError("voxelize_pack: voxel_feats is required with feats")
        _check_cuda_contiguous(voxel_feats, "voxel_feats")
        _check_float(voxel_feats, "voxel_feats")
        C = feats.shape[1]
        if feats.shape[0] != n or voxel_feats.shape[0] < n or voxel_feats.shape[1] != C:
            raise RuntimeError("voxelize_pack: feats (N,C) / voxel_feats (N,C) do not match the points")
    dev, stream = _where(points)
    ws, wp, wn = _ws_args(_lib.lib().v3d_grid_subsample_workspace_bytes(lengths.shape[0], n, C), points)
    rc = _lib.lib().v3d_voxelize_pack_f32(
        points.data_ptr(), lengths.data_ptr(), _ptr(feats) if C else None, C, voxels.data_ptr(), nodes.data_ptr(),
        _ptr(voxel_feats) if C else None, voxel_lengths.data_ptr(), num_voxels.data_ptr(), lengths.shape[0], n,
        float(voxel_size), wp, wn, dev, stream)
    _lib.check(rc, "voxelize_pack_mode")


# --------------------------------------------------------------------------------------------------------
# Correspondence selectors: pure torch in the reference (ops/mutual_topk_select.py).
# --------------------------------------------------------------------------------------------------------
SEL_LARGEST, SEL_MUTUAL, SEL_THRESHOLD, SEL_DUSTBIN = 1, 2, 4, 8


def _check_bool(t, name):
    if t.dtype != torch.bool:
        raise RuntimeError(f"{name} must be a bool tensor")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _select_flags(largest, mutual, threshold):
    return ((SEL_LARGEST if largest else 0) | (SEL_MUTUAL if mutual else 0)
            | (SEL_THRESHOLD if threshold is not None else 0))


def _select_outputs(name, corr_mat, out_batch, out_row, out_col, out_score, num_out, shape):
    capacity = None
    for t, n in ((out_batch, "out_batch"), (out_row, "out_row"), (out_col, "out_col")):
        if t is not None:
            _check_cuda_contiguous(t, n)
            _check_long(t, n)
            capacity = t.numel() if capacity is None else min(capacity, t.numel())
    if out_score is not None:
        _check_cuda_contiguous(out_score, "out_score")
        _check_float(out_score, "out_score")
        capacity = out_score.numel() if capacity is None else min(capacity, out_score.numel())
    if num_out is not None:
        _check_cuda_contiguous(num_out, "num_out")
        _check_long(num_out, "num_out")
    if corr_mat is not None:
        _check_cuda_contiguous(corr_mat, "corr_mat")
        _check_bool(corr_mat, "corr_mat")
        if tuple(corr_mat.shape) != tuple(shape):
            raise RuntimeError(f"{name}: corr_mat must have shape {tuple(shape)}")
    return capacity or 0


def mutual_topk_select(score_mat, k, corr_mat=None, out_batch=None, out_row=None, out_col=None, out_score=None,
                       num_out=None, row_masks=None, col_masks=None, largest=True, threshold=None, mutual=True):
    """score_mat (B,N,M) fp32 -> corr_mat (B,N,M) bool and/or compacted (batch,row,col,score) + device count."""
    _check_cuda_contiguous(score_mat, "score_mat")
    _check_float(score_mat, "score_mat")
    B, N, M = score_mat.shape
    for t, n, shape in ((row_masks, "row_masks", (B, N)), (col_masks, "col_masks", (B, M))):
        if t is not None:
            _check_cuda_contiguous(t, n)
            _check_bool(t, n)
            if tuple(t.shape) != shape:
                raise RuntimeError(f"mutual_topk_select: {n} must have shape {shape}")
    capacity = _select_outputs("mutual_topk_select", corr_mat, out_batch, out_row, out_col, out_score, num_out,
                               (B, N, M))
    dev, stream = _where(score_mat)
    ws, wp, wn = _ws_args(_lib.lib().v3d_mutual_topk_select_workspace_bytes(B, N, M, int(k)), score_mat)
    rc = _lib.lib().v3d_mutual_topk_select_f32(
        score_mat.data_ptr(), _ptr(row_masks), _ptr(col_masks), B, N, M, int(k),
        _select_flags(largest, mutual, threshold), float(threshold if threshold is not None else 0.0), _ptr(corr_mat),
        _ptr(out_batch), _ptr(out_row), _ptr(out_col), _ptr(out_score), _ptr(num_out), capacity, wp, wn, dev, stream)
    _lib.check(rc, "mutual_topk_select")


def mutual_select_lists(row_idx, row_val, col_idx, col_val, num_cols_total, corr_mat=None, out_batch=None,
                        out_row=None, out_col=None, out_score=None, num_out=None, row_masks=None, col_masks=None,
                        largest=False, threshold=None, mutual=True):
    """row_idx/row_val (B,N,k), col_idx/col_val (B,M,k) top-k lists of both sides -> same outputs as above."""
    for t, n in ((row_idx, "row_idx"), (col_idx, "col_idx")):
        _check_cuda_contiguous(t, n)
        _check_long(t, n)
    for t, n in ((row_val, "row_val"), (col_val, "col_val")):
        if t is not None:
            _check_cuda_contiguous(t, n)
            _check_float(t, n)
    B, N, k = row_idx.shape
    M = col_idx.shape[1]
    if M != int(num_cols_total) or col_idx.shape[0] != B or col_idx.shape[2] != k:
        raise RuntimeError("mutual_select_lists: row lists (B,N,k) and column lists (B,M,k) do not match")
    for t, n in ((row_masks, "row_masks"), (col_masks, "col_masks")):
        if t is not None:
            _check_cuda_contiguous(t, n)
            _check_bool(t, n)
    capacity = _select_outputs("mutual_select_lists", corr_mat, out_batch, out_row, out_col, out_score, num_out,
                               (B, N, M))
    dev, stream = _where(row_idx)
    ws, wp, wn = _ws_args(_lib.lib().v3d_mutual_select_lists_workspace_bytes(B, N, M, int(k)), row_idx)
    rc = _lib.lib().v3d_mutual_select_lists_f32(
        row_idx.data_ptr(), _ptr(row_val), col_idx.data_ptr(), _ptr(col_val), _ptr(row_masks), _ptr(col_masks), B, N, M,
        k, _select_flags(largest, mutual, threshold), float(threshold if threshold is not None else 0.0),
        _ptr(corr_mat), _ptr(out_batch), _ptr(out_row), _ptr(out_col), _ptr(out_score), _ptr(num_out), capacity, wp, wn,
        dev, stream)
    _lib.check(rc, "mutual_select_lists")


def _matrix_select_outputs(out_row, out_col, out_score, num_out):
    capacity = _select_outputs("select", None, None, out_row, out_col, out_score, num_out, ())
    return capacity


def threshold_select(score_mat, threshold, out_row=None, out_col=None, out_score=None, num_out=None, largest=True):
    """score_mat (N,M) fp32 -> the cells with score > threshold (< if not largest) in nonzero order + device count."""
    _check_cuda_contiguous(score_mat, "score_mat")
    _check_float(score_mat, "score_mat")
    if score_mat.dim() != 2:
        raise RuntimeError("threshold_select: score_mat must be a 2-D tensor")
    if num_out is None:
        raise RuntimeError("threshold_select: num_out is required")
    capacity = _matrix_select_outputs(out_row, out_col, out_score, num_out)
    N, M = score_mat.shape
    dev, stream = _where(score_mat)
    ws, wp, wn = _ws_args(_lib.lib().v3d_threshold_select_workspace_bytes(N, M), score_mat)
    rc = _lib.lib().v3d_threshold_select_f32(
        score_mat.data_ptr(), N, M, float(threshold), SEL_LARGEST if largest else 0, _ptr(out_row), _ptr(out_col),
        _ptr(out_score), _ptr(num_out), capacity, wp, wn, dev, stream)
    _lib.check(rc, "threshold_select")


def global_topk_select(score_mat, k, out_row=None, out_col=None, out_score=None, num_out=None, largest=True,
                       has_dustbin=False):
    """score_mat (N,M) fp32 -> the k best cells of the flattened matrix, best first (ties: lower flat index)."""
    _check_cuda_contiguous(score_mat, "score_mat")
    _check_float(score_mat, "score_mat")
    if score_mat.dim() != 2:
        raise RuntimeError("global_topk_select: score_mat must be a 2-D tensor")
    if has_dustbin and num_out is None:
        raise RuntimeError("global_topk_select: num_out is required with has_dustbin")
    capacity = _matrix_select_outputs(out_row, out_col, out_score, num_out)
    N, M = score_mat.shape
    dev, stream = _where(score_mat)
    ws, wp, wn = _ws_args(_lib.lib().v3d_global_topk_select_workspace_bytes(N, M, int(k)), score_mat)
    rc = _lib.lib().v3d_global_topk_select_f32(
        score_mat.data_ptr(), N, M, int(k), (SEL_LARGEST if largest else 0) | (SEL_DUSTBIN if has_dustbin else 0),
        _ptr(out_row), _ptr(out_col), _ptr(out_score), _ptr(num_out), capacity, wp, wn, dev, stream)
    _lib.check(rc, "global_topk_select")


# --------------------------------------------------------------------------------------------------------
# PACK-mode row gathers: pure torch in the reference (ops/index_select.py, ops/pooling.py,
# ops/nearest_interpolate.py, ops/knn_interpolate.py).  Features (N,C) row-major, tables (M,K) int64, index N = none.
# --------------------------------------------------------------------------------------------------------
def index_select_rows(sources, indices, targets, index_stride=1):
    """targets[l,:] = sources[indices.view(-1)[l*index_stride],:] (zeros outside [0,N)); any dtype, 2-D sources."""
    _check_cuda_contiguous(sources, "sources")
    _check_cuda_contiguous(indices, "indices")
    _check_cuda_contiguous(targets, "targets")
    _check_long(indices, "indices")
    _same_dtype("index_select_rows", sources, targets)
    N, row_bytes = sources.shape[0], sources.shape[1] * sources.element_size()
    L = targets.numel() // max(sources.shape[1], 1)
    if indices.numel() < (L - 1) * int(index_stride) + 1 and L > 0:
        raise RuntimeError("index_select_rows: indices too short for the requested rows")
    dev, stream = _where(sources)
    _lib.check(_lib.lib().v3d_index_select_rows(sources.data_ptr(), indices.data_ptr(), int(index_stride),
                                                targets.data_ptr(), L, N, row_bytes, dev, stream), "index_select_rows")


def local_maxpool_pack(feats, neighbor_indices, pooled, argk=None):
    """feats (N,C) fp32, neighbor_indices (M,K) -> pooled (M,C); argk (M,C) uint8 = first maximising column."""
    for t, n in ((feats, "feats"), (pooled, "pooled")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(neighbor_indices, "neighbor_indices")
    _check_long(neighbor_indices, "neighbor_indices")
    if argk is not None:
        _check_cuda_contiguous(argk, "argk")
        if argk.dtype != torch.uint8:
            raise RuntimeError("argk must be a byte tensor")
    M, K = neighbor_indices.shape
    N, C = feats.shape
    dev, stream = _where(feats)
    _lib.check(_lib.lib().v3d_local_maxpool_pack_f32(feats.data_ptr(), neighbor_indices.data_ptr(), pooled.data_ptr(),
                                                     _ptr(argk), M, N, K, C, dev, stream), "local_maxpool_pack_mode")


def knn_interp_weights_pack(q_points, s_points, neighbor_indices, weights, eps):
    """q (M,3), s (N,3) fp32, table (M,K) -> weights (M,k_used), k_used = weights.shape[1] <= K."""
    for t, n in ((q_points, "q_points"), (s_points, "s_points"), (weights, "weights")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(neighbor_indices, "neighbor_indices")
    _check_long(neighbor_indices, "neighbor_indices")
    M, K = neighbor_indices.shape
    dev, stream = _where(q_points)
    _lib.check(_lib.lib().v3d_knn_interp_weights_pack_f32(
        q_points.data_ptr(), s_points.data_ptr(), neighbor_indices.data_ptr(), weights.data_ptr(), M,
        s_points.shape[0], K, weights.shape[1], float(eps), dev, stream), "knn_interpolate_pack_mode")


def rows_weighted_sum(feats, neighbor_indices, weights, out):
    """out[m,:] = sum_k weights[m,k] * padded_feats[neighbor_indices[m,k],:], k < weights.shape[1]."""
    for t, n in ((feats, "feats"), (weights, "weights"), (out, "out")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(neighbor_indices, "neighbor_indices")
    _check_long(neighbor_indices, "neighbor_indices")
    M, K = neighbor_indices.shape
    N, C = feats.shape
    dev, stream = _where(feats)
    _lib.check(_lib.lib().v3d_rows_weighted_sum_f32(feats.data_ptr(), neighbor_indices.data_ptr(), weights.data_ptr(),
                                                    out.data_ptr(), M, N, K, weights.shape[1], C, dev, stream),
               "rows_weighted_sum")


def global_avgpool_pack(feats, lengths, pooled):
    """feats (N,C) fp32, lengths (B,) int64 on the device -> pooled (B,C)."""
    for t, n in ((feats, "feats"), (pooled, "pooled")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(lengths, "lengths")
    _check_long(lengths, "lengths")
    dev, stream = _where(feats)
    _lib.check(_lib.lib().v3d_global_avgpool_pack_f32(feats.data_ptr(), lengths.data_ptr(), pooled.data_ptr(),
                                                      lengths.shape[0], feats.shape[1], dev, stream),
               "global_avgpool_pack_mode")


def rows_csr_build(indices, num_sources):
    """Inverse (CSR over sources) of a neighbour table; returns the opaque device buffer the scatter calls take."""
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    L, N = indices.numel(), int(num_sources)
    nbytes = _lib.lib().v3d_rows_csr_bytes(N, L)
    csr = _workspace(nbytes, indices)
    dev, stream = _where(indices)
    _lib.check(_lib.lib().v3d_rows_csr_build(indices.data_ptr(), L, N, csr.data_ptr(), csr.numel(), dev, stream),
               "rows_csr_build")
    return csr


def rows_scatter(target_grads, csr, source_grads, table_shape, mode=0, weights=None, argk=None):
    """Atomic-free backward of the row gathers; table_shape = (M, K) of the table the csr was built from."""
    for t, n in ((target_grads, "target_grads"), (source_grads, "source_grads")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    M, K = table_shape
    N, C = source_grads.shape
    k_used = weights.shape[1] if (weights is not None and mode == 1) else K
    dev, stream = _where(target_grads)
    _lib.check(_lib.lib().v3d_rows_scatter_f32(target_grads.data_ptr(), csr.data_ptr(), _ptr(weights), _ptr(argk),
                                               int(mode), source_grads.data_ptr(), M * K, N, K, k_used, C, dev, stream),
               "rows_scatter")


# --------------------------------------------------------------------------------------------------------
# Fused grouping of the batch-mode layers: group_gather + subtract + cat in the reference.
# --------------------------------------------------------------------------------------------------------
def sa_group(q_points, s_points, s_feats, indices, grouped):
    """q_points (B,3,M), s_points (B,3,N), s_feats (B,C,N) or None, indices (B,M,K) -> grouped (B,C+3,M,K)."""
    tensors = [(q_points, "q_points"), (s_points, "s_points"), (grouped, "grouped")]
    if s_feats is not None:
        tensors.append((s_feats, "s_feats"))
    for t, n in tensors:
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    B, _, N = s_points.shape
    M, K = indices.shape[1], indices.shape[2]
    C = s_feats.shape[1] if s_feats is not None else 0
    if q_points.shape[1] != 3 or s_points.shape[1] != 3 or tuple(grouped.shape) != (B, C + 3, M, K):
        raise RuntimeError("sa_group: expected q_points (B,3,M), s_points (B,3,N), grouped (B,C+3,M,K)")
    dev, stream = _where(s_points)
    _lib.check(_lib.lib().v3d_sa_group_f32(q_points.data_ptr(), s_points.data_ptr(), _ptr(s_feats), indices.data_ptr(),
                                           grouped.data_ptr(), B, C, N, M, K, dev, stream), "sa_group")


def edge_group(q_feats, s_feats, indices, grouped):
    """q_feats (B,C,M), s_feats (B,C,N), indices (B,M,K) -> grouped (B,2C,M,K) = cat([q, neighbours - q])."""
    for t, n in ((q_feats, "q_feats"), (s_feats, "s_feats"), (grouped, "grouped")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(indices, "indices")
    _check_long(indices, "indices")
    B, C, N = s_feats.shape
    M, K = indices.shape[1], indices.shape[2]
    if tuple(q_feats.shape) != (B, C, M) or tuple(grouped.shape) != (B, 2 * C, M, K):
        raise RuntimeError("edge_group: expected q_feats (B,C,M), grouped (B,2C,M,K)")
    dev, stream = _where(s_feats)
    _lib.check(_lib.lib().v3d_edge_group_f32(q_feats.data_ptr(), s_feats.data_ptr(), indices.data_ptr(),
                                             grouped.data_ptr(), B, C, N, M, K, dev, stream), "edge_group")


def kpconv_gather(q_points, s_points, s_feats, neighbor_indices, kernel_points, weighted_feats, neighbor_num, sigma):
    """KPConv aggregation: weighted_feats (M,K,C) and (optional) neighbor_num (M,) int64; see include/v3d_hip.h."""
    for t, n in ((q_points, "q_points"), (s_points, "s_points"), (s_feats, "s_feats"),
                 (kernel_points, "kernel_points"), (weighted_feats, "weighted_feats")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(neighbor_indices, "neighbor_indices")
    _check_long(neighbor_indices, "neighbor_indices")
    if neighbor_num is not None:
        _check_cuda_contiguous(neighbor_num, "neighbor_num")
        _check_long(neighbor_num, "neighbor_num")
    M, H = neighbor_indices.shape
    N, C = s_feats.shape
    K = kernel_points.shape[0]
    if tuple(weighted_feats.shape) != (M, K, C) or q_points.shape[0] != M or s_points.shape[0] != N:
        raise RuntimeError("kpconv_gather: expected q_points (M,3), s_points (N,3), weighted_feats (M,K,C)")
    dev, stream = _where(s_feats)
    ws = _workspace(_lib.lib().v3d_kpconv_gather_workspace_bytes(N), s_feats) if neighbor_num is not None else None
    rc = _lib.lib().v3d_kpconv_gather_f32(
        q_points.data_ptr(), s_points.data_ptr(), s_feats.data_ptr(), neighbor_indices.data_ptr(),
        kernel_points.data_ptr(), weighted_feats.data_ptr(), _ptr(neighbor_num), M, N, H, K, C, float(sigma), _ptr(ws),
        ws.numel() if ws is not None else 0, dev, stream)
    _lib.check(rc, "kpconv_gather")


def point_to_node_partition(points, nodes, point_to_node, node_sizes=None, node_masks=None, max_size=None):
    """points (N,3), nodes (M,3) fp32 -> point_to_node (N) int64 [+ node_sizes (M) int64, node_masks (M) bool, max_size ()].
    Returns the workspace that ``point_to_node_knn`` consumes."""
    for t, n in ((points, "points"), (nodes, "nodes")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    for t, n in ((point_to_node, "point_to_node"), (node_sizes, "node_sizes"), (max_size, "max_size")):
        if t is not None:
            _check_cuda_contiguous(t, n)
            _check_long(t, n)
    if node_masks is not None:
        _check_cuda_contiguous(node_masks, "node_masks")
        _check_bool(node_masks, "node_masks")
    N, M = points.shape[0], nodes.shape[0]
    ws = _workspace(_lib.lib().v3d_point_to_node_workspace_bytes(N, M), points)
    dev, stream = _where(points)
    _lib.check(_lib.lib().v3d_point_to_node_partition_f32(
        points.data_ptr(), nodes.data_ptr(), N, M, point_to_node.data_ptr(), _ptr(node_sizes), _ptr(node_masks),
        _ptr(max_size), ws.data_ptr(), ws.numel(), dev, stream), "point_to_node_partition")
    return ws


def point_to_node_knn(workspace, num_points, node_knn_indices, node_knn_masks=None):
    """node_knn_indices (M,K) int64 / node_knn_masks (M,K) bool from the workspace of ``point_to_node_partition``."""
    _check_cuda_contiguous(node_knn_indices, "node_knn_indices")
    _check_long(node_knn_indices, "node_knn_indices")
    if node_knn_masks is not None:
        _check_cuda_contiguous(node_knn_masks, "node_knn_masks")
        _check_bool(node_knn_masks, "node_knn_masks")
    M, K = node_knn_indices.shape
    dev, stream = _where(node_knn_indices)
    _lib.check(_lib.lib().v3d_point_to_node_knn(workspace.data_ptr(), int(num_points), M, K, node_knn_indices.data_ptr(),
                                                _ptr(node_knn_masks), dev, stream), "point_to_node_partition")


def kpconv_gather_backward(q_points, s_points, neighbor_indices, kernel_points, grad_weighted, grad_neighbors, sigma):
    """grad_weighted (M,K,C) -> grad_neighbors (M,H,C) = influences^T x grad_weighted (then ``rows_scatter`` mode 0)."""
    for t, n in ((q_points, "q_points"), (s_points, "s_points"), (kernel_points, "kernel_points"),
                 (grad_weighted, "grad_weighted"), (grad_neighbors, "grad_neighbors")):
        _check_cuda_contiguous(t, n)
        _check_float(t, n)
    _check_cuda_contiguous(neighbor_indices, "neighbor_indices")
    _check_long(neighbor_indices, "neighbor_indices")
    M, H = neighbor_indices.shape
    K, C = grad_weighted.shape[1], grad_weighted.shape[2]
    if tuple(grad_neighbors.shape) != (M, H, C) or grad_weighted.shape[0] != M or kernel_points.shape[0] != K:
        raise RuntimeError("kpconv_gather_backward: expected grad_weighted (M,K,C), grad_neighbors (M,H,C)")
    dev, stream = _where(grad_weighted)
    _lib.check(_lib.lib().v3d_kpconv_gather_bwd_f32(
        q_points.data_ptr(), s_points.data_ptr(), neighbor_indices.data_ptr(), kernel_points.data_ptr(),
        grad_weighted.data_ptr(), grad_neighbors.data_ptr(), M, s_points.shape[0], H, K, C, float(sigma), dev, stream),
        "kpconv_gather_backward")


# --------------------------------------------------------------------------------------------------------
# Transformer layers over packs (no counterpart in the reference's extension: its layers call torch).
# --------------------------------------------------------------------------------------------------------
_ELEMENTS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # V3D_F32, V3D_F16, V3D_BF16


def _element(t, name):
    try:
        return _ELEMENTS[t.dtype]
    except KeyError:
        raise RuntimeError(f'"{name}" not implemented for \'{_TYPE_NAMES.get(t.dtype, t.dtype)}\'') from None


def _same_device(name, ref, *others):
    dev = ref.get_device()
    for o in others:
        if o is not None and o.get_device() != dev:
            raise RuntimeError(f"{name}: all tensors must be on one device, got {ref.device} and {o.device}")


def _operand(name, t, arg, shape, dtype=None):
    """An optional contiguous CUDA tensor of one shape and, if given, one element type."""
    if t is None:
        return
    _check_cuda_contiguous(t, arg)
    if t.shape != shape:
        raise RuntimeError(f"{name}: {arg} must have shape {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name}: expected scalar type {_TYPE_NAMES.get(dtype, dtype)} but found "
                           f"{_TYPE_NAMES.get(t.dtype, t.dtype)}")


def _layer_norm_check(name, feats, residual, weight, bias, stats):
    _check_cuda_contiguous(feats, "feats")
    if feats.dim() != 2:
        raise RuntimeError(f"{name}: feats must have shape (N, C)")
    shape = feats.shape
    _operand(name, residual, "residual", shape, feats.dtype)
    _operand(name, weight, "weight", shape[1:])
    _operand(name, bias, "bias", shape[1:], None if weight is None else weight.dtype)
    _operand(name, stats, "stats", (2, shape[0]), torch.float32)
    affine = bias if weight is None else weight
    return _element(feats, name), _element(feats if affine is None else affine, name), shape[0], shape[1]


def layer_norm_forward(feats, residual, weight, bias, targets, stats, eps):
    """targets (N, C) = layer norm of ``feats`` (+ ``residual``); ``stats`` (2, N) fp32 = mean and rstd of the rows, or
    None; see include/v3d_hip.h."""
    name = "layer_norm_forward"
    dtype, wdtype, rows, channels = _layer_norm_check(name, feats, residual, weight, bias, stats)
    _operand(name, targets, "targets", feats.shape, feats.dtype)
    _same_device(name, feats, residual, weight, bias, targets, stats)
    mean = _ptr(stats)
    dev, stream = _where(feats)
    rc = _lib.lib().v3d_layer_norm_fwd(feats.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), targets.data_ptr(), mean,
                                       None if mean is None else mean + 4 * rows, dtype, wdtype, rows, channels,
                                       float(eps), dev, stream)
    if rc != 0:
        _lib.check(rc, name)


def layer_norm_backward(target_grads, feats, residual, weight, stats, feats_grads, weight_grads, bias_grads):
    """The gradients of ``layer_norm_forward``: each of the three outputs may be None (not wanted)."""
    name = "layer_norm_backward"
    sums = weight_grads if weight_grads is not None else bias_grads
    _layer_norm_check(name, feats, residual, weight, None, stats)
    _operand(name, target_grads, "target_grads", feats.shape, feats.dtype)
    _operand(name, feats_grads, "feats_grads", feats.shape, feats.dtype)
    if sums is not None:
        dtype = sums.dtype if weight is None else weight.dtype
        _operand(name, weight_grads, "weight_grads", feats.shape[1:], dtype)
        _operand(name, bias_grads, "bias_grads", feats.shape[1:], dtype)
        _element(sums, name)
    _same_device(name, feats, target_grads, residual, weight, stats, feats_grads, weight_grads, bias_grads)
    _layer_norm_backward(target_grads, feats, residual, weight, stats, feats_grads, weight_grads, bias_grads)


def _layer_norm_backward(target_grads, feats, residual, weight, stats, feats_grads, weight_grads, bias_grads):
    """The launch alone, for the autograd function, whose tensors the forward has checked or the backward has made."""
    rows, channels = feats.shape
    sums = weight_grads if weight_grads is not None else bias_grads
    affine = weight if sums is None else sums
    lib = _lib.lib()
    ws, wp, wn = _ws_args(0 if sums is None else lib.v3d_layer_norm_bwd_workspace_bytes(rows, channels), feats)
    mean = stats.data_ptr()
    dev, stream = _where(feats)
    rc = lib.v3d_layer_norm_bwd(target_grads.data_ptr(), feats.data_ptr(), _ptr(residual), _ptr(weight), mean,
                                mean + 4 * rows, _ptr(feats_grads), _ptr(weight_grads), _ptr(bias_grads),
                                _ELEMENTS[feats.dtype], _ELEMENTS[(feats if affine is None else affine).dtype], rows,
                                channels, wp, wn, dev, stream)
    if rc != 0:
        _lib.check(rc, "layer_norm_backward")


def _heads(name, t, arg, dims, dtype):
    """(strides, shape) of features (.., heads, D) of any strides but the last, which is 1; 0 where there is one entry."""
    if not t.is_cuda:
        raise RuntimeError(f"{arg} must be a CUDA tensor")
    shape, strides = t.shape, t.stride()
    if len(shape) != dims:
        raise RuntimeError(f"{name}: {arg} must have {dims} dimensions, got {len(shape)}")
    if shape[-1] > 1 and strides[-1] != 1:
        raise RuntimeError(f"{name}: the last dimension of {arg} must be contiguous")
    if t.dtype != dtype:
        raise RuntimeError(f"{name}: expected scalar type {_TYPE_NAMES.get(dtype, dtype)} but found "
                           f"{_TYPE_NAMES.get(t.dtype, t.dtype)}")
    if 1 in shape:
        strides = [0 if n == 1 else s for n, s in zip(shape, strides)]
    return strides, shape


def _lengths(name, t, arg, count):
    _check_cuda_contiguous(t, arg)
    _check_long(t, arg)
    if t.shape != (count,):
        raise RuntimeError(f"{name}: {arg} must have shape {(count,)}")


_Strides6, _Strides8 = ctypes.c_int64 * 6, ctypes.c_int64 * 8


def _attention_check(name, q, k, v, q_lengths, s_lengths):
    qs, qshape = _heads(name, q, "q_feats", 3, q.dtype)
    ks, kshape = _heads(name, k, "k_feats", 3, q.dtype)
    vs, vshape = _heads(name, v, "v_feats", 3, q.dtype)
    if vshape != kshape or kshape[2] != qshape[2]:
        raise RuntimeError(f"{name}: expected q_feats (N, H, D), k_feats and v_feats (M, KV, D)")
    count = q_lengths.numel()
    _lengths(name, q_lengths, "q_lengths", count)
    _lengths(name, s_lengths, "s_lengths", count)
    sizes = (count, qshape[0], kshape[0], qshape[1], kshape[1], qshape[2])  # B, N, M, H, KV, D
    return _element(q, name), sizes, _Strides6(qs[0], qs[1], ks[0], ks[1], vs[0], vs[1])


def attention_pack_forward(q_feats, k_feats, v_feats, q_lengths, s_lengths, targets, lse, scale, causal, rest=None):
    """targets (N, H, D) = attention of ``q_feats`` (N, H, D) over ``k_feats`` / ``v_feats`` (M, KV, D) inside every
    sequence of the pack; for the backward: ``lse`` (N, H) fp32 and, of 16-bit types, ``rest`` (N, H, D) = what rounding took
    from ``targets``; see include/v3d_hip.h."""
    name = "attention_pack_forward"
    dtype, sizes, strides = _attention_check(name, q_feats, k_feats, v_feats, q_lengths, s_lengths)
    shape = q_feats.shape
    _operand(name, targets, "targets", shape, q_feats.dtype)
    _operand(name, lse, "lse", shape[:2], torch.float32)
    _operand(name, rest, "rest", shape, q_feats.dtype)
    _same_device(name, q_feats, k_feats, v_feats, q_lengths, s_lengths, targets, lse, rest)
    lib = _lib.lib()
    ws, wp, wn = _ws_args(lib.v3d_attention_pack_workspace_bytes(*sizes), q_feats)
    dev, stream = _where(q_feats)
    _lib.check(lib.v3d_attention_pack_fwd(q_feats.data_ptr(), k_feats.data_ptr(), v_feats.data_ptr(),
                                          q_lengths.data_ptr(), s_lengths.data_ptr(), targets.data_ptr(), _ptr(rest),
                                          _ptr(lse), dtype, *sizes, strides, scale, bool(causal), wp, wn, dev, stream),
               name)


def attention_pack_backward(target_grads, q_feats, k_feats, v_feats, targets, lse, q_lengths, s_lengths, q_grads, k_grads,
                            v_grads, scale, causal, rest=None):
    """The gradients of ``attention_pack_forward``, from its inputs, ``targets``, ``lse`` and (16-bit types) ``rest``;
    ``q_grads``, or ``k_grads`` and ``v_grads`` together, may be None (not wanted)."""
    name = "attention_pack_backward"
    _attention_check(name, q_feats, k_feats, v_feats, q_lengths, s_lengths)
    shape, kshape = q_feats.shape, k_feats.shape
    _operand(name, target_grads, "target_grads", shape, q_feats.dtype)
    _operand(name, targets, "targets", shape, q_feats.dtype)
    _operand(name, lse, "lse", shape[:2], torch.float32)
    _operand(name, rest, "rest", shape, q_feats.dtype)
    _operand(name, q_grads, "q_grads", shape, q_feats.dtype)
    _operand(name, k_grads, "k_grads", kshape, q_feats.dtype)
    _operand(name, v_grads, "v_grads", kshape, q_feats.dtype)
    _same_device(name, q_feats, k_feats, v_feats, q_lengths, s_lengths, target_grads, targets, lse, rest, q_grads, k_grads,
                 v_grads)
    _attention_pack_backward(target_grads, q_feats, k_feats, v_feats, targets, lse, q_lengths, s_lengths, q_grads, k_grads,
                             v_grads, scale, causal, rest)


def _attention_pack_backward(target_grads, q, k, v, targets, lse, q_lengths, s_lengths, q_grads, k_grads, v_grads, scale,
                             causal, rest):
    """The launch alone, for the autograd function, whose tensors the forward has checked or the backward has made."""
    (N, H, D), (M, KV, _) = q.shape, k.shape
    B = q_lengths.shape[0]
    (qs, _), (ks, _), (vs, _) = (_heads("attention_pack_backward", t, "features", 3, q.dtype) for t in (q, k, v))
    lib = _lib.lib()
    ws, wp, wn = _ws_args(lib.v3d_attention_pack_bwd_workspace_bytes(B, N, M, H, KV, D), q)
    dev, stream = _where(q)
    rc = lib.v3d_attention_pack_bwd(target_grads.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), targets.data_ptr(),
                                    _ptr(rest), lse.data_ptr(), q_lengths.data_ptr(), s_lengths.data_ptr(),
                                    _ptr(q_grads), _ptr(k_grads), _ptr(v_grads), _ELEMENTS[q.dtype], B, N, M, H, KV, D,
                                    _Strides6(qs[0], qs[1], ks[0], ks[1], vs[0], vs[1]), scale, bool(causal), wp,
                                    wn, dev, stream)
    if rc != 0:
        _lib.check(rc, "attention_pack_backward")


def cached_attention(q_feats, k_cache, v_cache, lengths, targets, scale):
    """targets (B, T, H, D) = attention of the newest T tokens of every sequence over its cache (B, C, KV, D), of which
    ``lengths`` (B,) rows are filled; see include/v3d_hip.h."""
    name = "cached_attention"
    qs, shape = _heads(name, q_feats, "q_feats", 4, q_feats.dtype)
    ks, kshape = _heads(name, k_cache, "k_cache", 4, q_feats.dtype)
    vs, vshape = _heads(name, v_cache, "v_cache", 4, q_feats.dtype)
    _operand(name, targets, "targets", shape, q_feats.dtype)
    dtype = _element(q_feats, name)
    B, T, H, D = shape
    if kshape != vshape or kshape[0] != B or kshape[3] != D:
        raise RuntimeError(f"{name}: expected q_feats (B, T, H, D), k_cache and v_cache (B, C, KV, D)")
    if B > 1 and T > 1 and qs[0] != T * qs[1]:
        raise RuntimeError(f"{name}: the tokens of q_feats must be at one stride")
    _lengths(name, lengths, "lengths", B)
    _same_device(name, q_feats, k_cache, v_cache, lengths, targets)
    C, KV = kshape[1], kshape[2]
    strides = _Strides8(qs[1] if T > 1 else qs[0], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    lib = _lib.lib()
    ws, wp, wn = _ws_args(lib.v3d_cached_attention_workspace_bytes(B, T, C, H, KV, D), q_feats)
    dev, stream = _where(q_feats)
    _lib.check(lib.v3d_cached_attention(q_feats.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(),
                                        targets.data_ptr(), dtype, B, T, C, H, KV, D, strides, scale, wp, wn, dev,
                                        stream), name)


# --------------------------------------------------------------------------------------------------------
# The reference extension's NumPy (CPU) entry points that the pack-mode pyramid uses (csrc/pybind.cpp:34-70), so that
# `vision3d.array_ops` (collate-time neighbourhood construction) finds them on `vision3d.ext`: NumPy arrays in and out
# like the reference, the work done by the pack-mode GPU kernels above.  Differences from the CPU code are stated per
# function.  The deformation-graph / depth-image helpers (csrc/pybind.cpp:20-32, :52-61) are outside this path.
# --------------------------------------------------------------------------------------------------------
def _np_to_dev(a, dtype):
    import numpy as np

    return torch.from_numpy(np.ascontiguousarray(np.asarray(a), dtype=dtype)).cuda()


def radius_neighbors(q_points, s_points, q_lengths, s_lenghts, radius):
    """(total_q, max_count) int64 neighbour table, ascending by distance, padded with total_s
    (csrc/cpu/radius_neighbors/radius_neighbors.cpp:5-93; keyword `s_lenghts` as registered, pybind.cpp:41).

    Strict on ``radius - sqrt(d2) > 0`` (the count kernel's predicate: supports exactly AT the radius are left out; the
    table of the inclusive search kernel is cut at that count).  The CPU code's nanoflann search tests ``d2 < radius *
    radius`` in float (radius_neighbors.cpp:24,:60): the two predicates can disagree for a support within one ulp of the
    sphere -- that boundary case is parity unpinned (the oracle uses the sqrt form too).  Difference: the table is at most 512 wide (the
    search kernel's list); a query with more than 512 neighbours raises instead of widening it further."""
    import numpy as np

    q, s = _np_to_dev(q_points, np.float32), _np_to_dev(s_points, np.float32)
    ql, sl = _np_to_dev(q_lengths, np.int64), _np_to_dev(s_lenghts, np.int64)
    if q.shape[0] == 0:
        return np.zeros((0, 0), dtype=np.int64)
    counts = torch.empty((q.shape[0],), dtype=torch.long, device=q.device)
    radius_count_pack(q, s, ql, sl, counts, float(radius))  # strict: radius - d > 0
    filled = int(counts.max().item())
    if filled > 512:
        raise RuntimeError("radius_neighbors: a query has more than 512 neighbours; use radius_search_pack_mode with a limit")
    limit = next(w for w in (64, 128, 256, 512) if filled <= w)
    out = torch.empty((q.shape[0], limit), dtype=torch.long, device=q.device)
    radius_search_pack(q, s, ql, sl, out, float(radius), limit)
    # ascending by distance: what the inclusive search adds (d == radius) sits behind the strict neighbours
    keep = torch.arange(limit, device=q.device).unsqueeze(0) < counts.unsqueeze(1)
    out = torch.where(keep, out, torch.full_like(out, s.shape[0]))
    return out[:, :filled].cpu().numpy()


def grid_subsampling(points, lengths, voxel_size):
    """(sampled_points (M,3) float32, sampled_lengths (B,) int64) -- csrc/cpu/grid_subsampling/grid_subsampling.cpp:30-55.
    Voxel barycentres per cloud; rows come out ordered by (cloud, vx, vy, vz) where the CPU code emits its hash map's
    iteration order (unspecified): compare as sets."""
    import numpy as np

    p, ln = _np_to_dev(points, np.float32), _np_to_dev(lengths, np.int64)
    out = torch.empty_like(p)
    out_len = torch.empty_like(ln)
    num = torch.zeros((), dtype=torch.long, device=p.device)
    grid_subsample_pack(p, ln, out, out_len, num, float(voxel_size))
    m = int(num.item())
    if m < 0:
        raise RuntimeError("grid_subsampling: a cloud spans more than 2^18 voxels along an axis (or holds NaN)")
    return out[:m].cpu().numpy(), out_len.cpu().numpy()


def sample_nodes_with_fps(points, min_distance, num_samples):
    """Indices of furthest-point samples starting at point 0, until `num_samples` are taken (if > 0) or the furthest
    remaining point is closer than `min_distance` to the chosen set (csrc/cpu/node_sampling/node_sampling.cpp:10-77).

    Runs the batch FPS kernel and cuts the sequence where the selection distance first drops below `min_distance`.
    Among EQUALLY far candidates the kernel follows the CUDA kernel's order, the CPU code its swap-and-pop traversal: the
    two agree on tie-free clouds."""
    import numpy as np

    p = _np_to_dev(points, np.float32)
    n = p.shape[0]
    if n == 0:
        return np.zeros((0,), dtype=np.int64)
    want = n if num_samples is None or num_samples <= 0 else min(int(num_samples), n)
    take = want if min_distance is None or min_distance <= 0 else min(want, 1024)
    while True:
        dist = torch.full((1, n), 1e10, dtype=torch.float32, device=p.device)
        idx = torch.zeros((1, take), dtype=torch.long, device=p.device)
        furthest_point_sample(p.unsqueeze(0), dist, idx, take)
        host_idx = idx[0].cpu().numpy()  # the entry point returns NumPy: this copy is its one synchronisation per pass
        if min_distance is None or min_distance <= 0:
            return host_idx
        # selection distance of sample j = its distance to the nearest of the samples before it (float64, on the host:
        # the result is host-side anyway, and `take` <= 1024 on the first pass)
        chosen = np.asarray(points, dtype=np.float32)[host_idx].astype(np.float64)
        gaps = np.full((take,), np.inf)
        for j0 in range(0, take, 256):
            blk = chosen[j0:j0 + 256]
            d = np.sqrt(((blk[:, None, :] - chosen[None, :j0 + blk.shape[0], :]) ** 2).sum(-1))
            d[np.arange(blk.shape[0])[:, None] + j0 <= np.arange(d.shape[1])[None, :]] = np.inf  # earlier samples only
            gaps[j0:j0 + blk.shape[0]] = d.min(axis=1)
        below = np.nonzero(gaps.astype(np.float32) < np.float32(min_distance))[0]  # gaps[0] = inf: the first always stays
        if below.size:
            return host_idx[: int(below[0])]
        if take >= want:
            return host_idx
        take = min(want, take * 4)


def _outside_the_path(name):
    def stub(*_args, **_kwargs):
        raise NotImplementedError(
            f"vision3d.ext.{name} belongs to the reference's deformation-graph / depth-image CPU helpers "
            "(csrc/pybind.cpp:20-32, :52-61), which are outside the operator path this library replaces")

    stub.__name__ = name
    return stub


for _name in ("depth_to_mesh", "erode_mesh", "sample_nodes", "compute_edges_geodesic", "compute_edges_euclidean",
              "compute_pixel_anchors_geodesic", "node_and_edge_clean_up", "update_pixel_anchors", "compute_clusters",
              "build_deformation_graph_from_point_cloud"):
    globals()[_name] = _outside_the_path(_name)
del _name
