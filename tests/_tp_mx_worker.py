"""Worker of tests/test_gpu_mx_engine_paths.py: one of two tensor-parallel ranks, both on GPU 0, whose target has a block-scaled cache.  Writes the logits of
a verify step, its shard of the first layer's cache and its page table, and what the speculation of two models ends with."""
import os
import sys
from pathlib import Path

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tests import golden_cfg as gc  # noqa: E402


def main():
    from magicdec_amd import harness
    from magicdec_amd.Engine import model_core
    from magicdec_amd.Engine.SnapKV.backend import LMBackend
    from magicdec_amd.Engine.SnapKV.backend_draft import LMBackend_Draft
    from magicdec_amd.Engine.tp import init_dist
    ck, out = Path(os.environ["MD_CKPT"]), os.environ["MD_OUT"]
    gc.register_tiny(model_core)
    rank, group, dgroup = init_dist([0, 1])
    eng = LMBackend(dtype=torch.bfloat16, device="cuda:0", dec_len=gc.GAMMA + 1)
    eng.load_model(ck / "tinytgt" / "model.pth", use_tp=True, rank_group=[0, 1], group=group)
    eng.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, kv_dtype=os.environ["MD_KV_DTYPE"])
    drf = LMBackend_Draft(dtype=torch.bfloat16, device="cuda:0", draft_budget=gc.BUDGET)
    drf.load_model(ck / "tinytgt" / "model.pth", use_tp=True, rank_group=[0, 1], group=dgroup)
    drf.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, draft_budget=gc.BUDGET)
    ids = gc.synthetic_batches()[0].to("cuda:0")
    eng.encode(ids)
    cache = eng.model.layers[0].attention.kv_cache.kv_cache.cpu()
    eng.inference(ids[:, :gc.GAMMA + 1].clone())
    logits = eng.model._last_logits.float().cpu()
    st, _ = harness.run_longspec_batch(eng, drf, ids, gc.GAMMA, gc.MAX_LEN, gc.EOT_1, gc.EOT_2, barrier=dist.barrier)
    torch.save(dict(cache=cache, logits=logits, output=st.output.cpu(), num_nodes=st.num_nodes.cpu(), iters=st.iters), os.path.join(out, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()
    print(f"rank {rank}: OK", flush=True)


if __name__ == "__main__":
    main()
