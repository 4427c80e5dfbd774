"""B200-native (sm_100a) row-wise inference kernels behind the entry points of
fengwang/cuda-kernels-optimized-for-rtx5090: softmax.run, rmsnorm.run, rope.run and topk.run take and return the same
dicts as the reference's softmax/baseline.py and {rmsnorm,rope,topk}/candidate.py. The CUDA libraries are built in
tree by ckb200.build (lib/<op>/libkernel.so); there is no CPU fallback. ckb200.hostpipe.RowPipeline streams pinned
host batches through any of them with the copies overlapped. Beside them stand the rest of a drafted-decoding step:
attention.paged_attention reads the paged cache that rope writes, verify.verify_drafts checks drafted tokens against the target's probabilities.
"""

from . import attention, build, hostpipe, rmsnorm, rope, sharded, softmax, topk, verify  # noqa: F401

__all__ = ["attention", "build", "hostpipe", "rmsnorm", "rope", "sharded", "softmax", "topk", "verify"]
