"""Data-parallel distillation on the GPU (ranks may share one): every rank trains on its share of one batch. MLAPI_DP_FUSED=1
(default): the exchange runs inside the step's last kernel; 0: gradient, all-reduce and update apart; MLAPI_DP_TWO_SHOT=1:
owner ranks reduce and update, the others copy. OUT gets params and loss, named <world>_<rank><how>."""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", ".."))
from mlapi_amd.models.linear import LinearModel  # noqa: E402
from mlapi_amd.parallel.comm import init_distributed, shutdown  # noqa: E402
from mlapi_amd.train.softmax_sgd import SoftmaxSGDTrainer, synthetic_multiclass, teacher_top  # noqa: E402

info = init_distributed(use_gpu=True, comm="p2p")
dev, out, r, w = info.device, os.environ["OUT"], info.rank, info.world
fused = os.environ.get("MLAPI_DP_FUSED", "1") != "0"
how = ("" if fused else "_apart") + ("_two" if os.environ.get("MLAPI_DP_TWO_SHOT") == "1" else "")
n, F, K = 1024, 60, 23
X, y = synthetic_multiclass(n, F, K, seed=1, device=dev)
idx, t = teacher_top(LinearModel.random(F, K, seed=2), X, 6)
tr = SoftmaxSGDTrainer(F, K, info=info, lr=0.3, momentum=0.5, device=dev, temperature=2.0, alpha=0.6)
assert tr.dp_exchange == ("local" if w == 1 else ("fused-p2p" if fused else "rccl")), tr.dp_exchange
mine = slice(r * n // w, (r + 1) * n // w)
Xa, ym, top = tr.prepare(X)[mine], y[mine], (idx[mine], t[mine])
for _ in range(4):
    tr.step(Xa, ym, teacher=top)
np.save(f"{out}/params_{w}_{r}{how}.npy", tr.params.cpu().numpy())
np.save(f"{out}/loss_{w}_{r}{how}.npy", np.float64(tr.last_loss()))
info.comm.wait()
tr.check()
shutdown(info)
