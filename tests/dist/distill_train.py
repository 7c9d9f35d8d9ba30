"""Data-parallel distillation on the CPU: every rank trains on its share of one batch; OUT gets the parameters."""
import os

import numpy as np
import torch

from mlapi_amd.models.linear import LinearModel
from mlapi_amd.parallel.comm import init_distributed, shutdown
from mlapi_amd.train.softmax_sgd import SoftmaxSGDTrainer, synthetic_multiclass, teacher_top

info = init_distributed()
X, y = synthetic_multiclass(128, 20, 6, seed=1)
idx, t = teacher_top(LinearModel.random(20, 6, seed=2), X, 3)
mine = slice(info.rank * 128 // info.world, (info.rank + 1) * 128 // info.world)
tr = SoftmaxSGDTrainer(20, 6, info=info, lr=0.5, momentum=0.9, device=torch.device("cpu"), temperature=2.0, alpha=0.6)
Xa = tr.prepare(X[mine])
for _ in range(5):
    tr.step(Xa, y[mine], teacher=(idx[mine], t[mine]))
np.save(os.path.join(os.environ["OUT"], f"params_{info.world}_{info.rank}.npy"), tr.params.numpy())
np.save(os.path.join(os.environ["OUT"], f"loss_{info.world}_{info.rank}.npy"), np.float64(tr.last_loss()))
shutdown(info)
