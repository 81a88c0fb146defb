"""Dense SDF inference for meshing ("next" row N3): the query part of
`Mesher.query_points` (utils/mesher.py:38-163) as one fused HIP launch per chunk.  Marching cubes and
Open3D mesh handling stay with the reference (skimage / open3d, out of scope)."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib


def query_points(neural_points, sdf_mlp, config, coord, bs=None, query_sdf=True, query_sem=False, query_color=False,
                 query_mask=True, query_locally=False, mask_min_nn_count: int = 4, out_torch: bool = True, sem_mlp=None):
    """Same 4-tuple as the reference method: (sdf_pred [N], sem_pred [N] int64 or None, None, mc_mask [N]); `out_torch=False`
    returns numpy arrays.  `query_sem` asks `sem_mlp` for the class of each point (0 where it has no neighbour).  The colour head
    is outside the hot-path scope."""
    if query_color:
        raise NotImplementedError("colour queries are outside the hot-path scope")
    if query_sem and sem_mlp is None:
        raise RuntimeError("query_sem needs a semantic decoder")
    lib = _lib.load()
    bs = int(bs or config.infer_bs)
    n = coord.shape[0]
    dev = neural_points.neural_points.device
    sdf = torch.zeros(n, device=dev, dtype=torch.float32)
    nn_cnt = torch.zeros(n, device=dev, dtype=torch.int32)
    view, keep = neural_points._map_view(bool(query_locally))
    W1, b1, W2, b2 = sdf_mlp.flat_params()
    for i in range(math.ceil(n / bs)):
        x = coord[i * bs:(i + 1) * bs].to(dev, torch.float32).contiguous()
        m = x.shape[0]
        _lib.check(
            lib.clid_sdf_query(C.byref(view), _lib.ptr(W1), _lib.ptr(b1), _lib.ptr(W2), _lib.ptr(b2),
                               float(sdf_mlp.sdf_scale), _lib.ptr(x), m, sdf[i * bs:].data_ptr(),
                               nn_cnt[i * bs:].data_ptr(), _lib.stream()),
            "clid_sdf_query",
        )
    sdf_pred = sdf if query_sdf else None
    sem_pred = torch.zeros(n, device=dev, dtype=torch.int64) if query_sem else None
    for i in range(math.ceil(n / bs) if query_sem else 0):
        at = slice(i * bs, (i + 1) * bs)
        sem_pred[at] = torch.where(nn_cnt[at] >= 1, _labels(neural_points, sem_mlp, config, coord[at].to(dev, torch.float32), query_locally), 0)
    mc_mask = (nn_cnt >= mask_min_nn_count).to(torch.float32) if query_mask else None
    if not out_torch:
        sdf_pred = None if sdf_pred is None else sdf_pred.cpu().numpy().astype("float64")
        sem_pred = None if sem_pred is None else sem_pred.cpu().numpy()
        mc_mask = None if mc_mask is None else mc_mask.cpu().numpy().astype("float64")
    return sdf_pred, sem_pred, None, mc_mask


@torch.no_grad()
def _labels(neural_points, sem_mlp, config, coord, query_locally):
    """Classes of one chunk of points (utils/mesher.py:118-131)."""
    feature, _, weight, _, _ = neural_points.query_feature(coord, training_mode=False, query_locally=bool(query_locally))
    if config.weighted_first:
        return sem_mlp.sem_label(feature)
    return (sem_mlp.sem_label_prob(feature) * weight).sum(dim=1).argmax(dim=1)  # the neighbours' log-probabilities, blended


class Mesher:
    """`Mesher` with the reference's constructor and `query_points` signature (utils/mesher.py:20-47) for the part that is
    on the hot path: the dense SDF / mask query.  Marching cubes and mesh export need skimage / open3d and stay with the
    reference (out of scope): those methods raise."""

    def __init__(self, config, neural_points, decoders: dict):
        self.config = config
        self.silence = getattr(config, "silence", True)
        self.neural_points = neural_points
        self.sdf_mlp = decoders["sdf"]
        self.sem_mlp = decoders.get("semantic")
        self.color_mlp = decoders.get("color")
        self.device = config.device
        self.cur_device = self.device
        self.dtype = config.dtype

    def query_points(self, coord, bs, query_sdf=True, query_sem=False, query_color=False, query_mask=True,
                     query_locally=False, mask_min_nn_count: int = 4, out_torch: bool = False):
        """utils/mesher.py:38-163: (sdf_pred, sem_pred, color_pred, mc_mask)."""
        return query_points(self.neural_points, self.sdf_mlp, self.config, coord, bs, query_sdf, query_sem, query_color,
                            query_mask, query_locally, mask_min_nn_count, out_torch, self.sem_mlp)

    def recon_aabb_mesh(self, *args, **kwargs):
        raise NotImplementedError("marching cubes / mesh export (utils/mesher.py:371-667) need skimage + open3d: out of scope")

    mc_mesh = recon_aabb_mesh
