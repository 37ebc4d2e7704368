"""A pair-stack block with dropout, sharded over two CPU ranks (gloo), has the masks of the unsharded one: the same seed on all ranks
gives the same result and gradients as one rank that holds everything."""
import os
import tempfile

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from openfold3_triangle_kernel_b200 import dap
from oracle import sequence_oracle as so
from test_dap_gloo import WORLD, TorchStages, _attention_fn


def _dropout(x, p, seed, shared_dim, residual):
    return residual + torch.where(so.dropout_mask(x.shape, p, *seed, shared_dim), x / (1 - round(65536 * p) / 65536), 0.0)


def _worker(rank, init_file, results):
    dist.init_process_group("gloo", init_method=f"file://{init_file}", rank=rank, world_size=WORLD)
    try:
        from openfold3_triangle_kernel_b200.pair_block import pair_stack_block
        from oracle.pair_block_oracle import block_params
        n, c, heads = 8, 8, 2
        g = torch.Generator().manual_seed(5)
        z, dy = (torch.randn(1, n, n, c, generator=g, dtype=torch.float64) for _ in range(2))
        mask = torch.ones(1, n, n, dtype=torch.float64)
        params = block_params(c, heads, 4, 9, dtype=torch.float64)
        alone = [dist.new_group([r]) for r in range(WORLD)][rank]
        kw = dict(trimul_backend=TorchStages(), attention_fn=_attention_fn, dropout=0.25, dropout_fn=_dropout, seed=(11, 3))
        zl, zr = dap.shard_rows(z, 1).clone().requires_grad_(True), z.clone().requires_grad_(True)
        out = pair_stack_block(zl, dap.shard_rows(mask, 1), params, heads, group=dist.group.WORLD, **kw)
        out.backward(dap.shard_rows(dy, 1))
        ref = pair_stack_block(zr, mask, params, heads, group=alone, **kw)
        ref.backward(dy)
        # (the attention wrapper's layer norm runs in fp32)
        assert torch.allclose(dap.gather_rows(out.detach(), 1), ref.detach(), atol=2e-5, rtol=2e-5)
        assert torch.allclose(dap.gather_rows(zl.grad, 1), zr.grad, atol=2e-4, rtol=2e-4)
        results[rank] = "ok"
    except Exception as e:  # noqa: BLE001
        import traceback
        results[rank] = "".join(traceback.format_exception(e))
    finally:
        dist.destroy_process_group()


def test_sharded_block_has_the_masks_of_the_unsharded_one():
    with tempfile.TemporaryDirectory() as tmp, mp.Manager() as manager:
        results = manager.dict()
        mp.spawn(_worker, args=(os.path.join(tmp, "init"), results), nprocs=WORLD, join=True)
        assert dict(results) == {r: "ok" for r in range(WORLD)}
