"""Engines with a block-scaled full-context cache (setup_caches(kv_dtype="mxfp8" / "mxfp4")) on the GPU: the operators of a step run together as a
user's program has them -- rows quantised behind the rotation, attention over them, the SnapKV select of rows read back, captured steps."""
import os
import tempfile

import pytest
import torch

from tests import golden_cfg as gc
from tests import mx_util as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ckpt_dir():
    from magicdec_amd.Engine import model_core
    d = tempfile.mkdtemp(prefix="md_mx_ckpt_")
    for name in gc.TINY:
        cfg, sd = gc.tiny(name)
        os.makedirs(os.path.join(d, name), exist_ok=True)
        torch.save(sd, os.path.join(d, name, "model.pth"))
        model_core.transformer_configs[name] = gc.config_kwargs(cfg)
    return d


def engine(ckpt_dir, kv_dtype, graphs=False, draft=True, cls=None, **more):
    from magicdec_amd.Engine.SnapKV.backend import LMBackend
    eng = (cls or LMBackend)(dtype=BF, device=DEV, dec_len=gc.GAMMA + 1, **(dict(draft_dec_len=1) if draft else {}))
    eng.load_model(os.path.join(ckpt_dir, "tinytgt", "model.pth"), use_tp=False)
    if graphs:
        eng.compile()
    eng.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, kv_dtype=kv_dtype, **(dict(draft_budget=gc.BUDGET) if draft else {}), **more)
    return eng


def quantized_step_error(eng, ref):
    """Logits of a verify step of `eng`, relative to those of `ref` (2-norms)."""
    return ((eng - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("kv_dtype", ["mxfp8", "mxfp4"])
def test_self_speculation_over_block_scaled_pages(ckpt_dir, kv_dtype):
    """The cache holds what the format says of the rows that a 16-bit engine appends in its first layer; the SnapKV draft gets rows of it; the
    loop generates, with captured steps bit for bit as without.  An element is off by 2^-4 (e4m3) or 1/4 (e2m1) of itself at most: logits
    of a step are held to as much of theirs, in 2-norm."""
    from magicdec_amd import harness
    ids = next(iter(gc.synthetic_batches())).to(DEV)
    logits, outs, caches = {}, {}, {}
    for kvd, graphs in (("bf16", False), (kv_dtype, False), (kv_dtype, True)):
        eng = engine(ckpt_dir, kvd, graphs)
        eng.encode(ids)
        kvc = eng.model.layers[0].attention.kv_cache
        if not graphs:
            caches[kvd] = (kvc.kv_cache.cpu().clone(), kvc.draft_cache.cpu().clone())
        eng.verify(ids[:, :gc.GAMMA + 1].clone())
        logits[(kvd, graphs)] = eng.model._last_logits.float().cpu()
        st, _ = harness.run_selfspec_batch(eng, ids, gc.GAMMA, gc.MAX_LEN, gc.EOT_1, gc.EOT_2, False)
        outs[(kvd, graphs)] = st
        assert st.iters > 0 and (st.num_nodes.cpu() > ids.shape[1]).all()
    D = caches["bf16"][0].shape[-1]
    pages = -(-ids.shape[1] // 128)
    code, scale = mx.unpack(caches[kv_dtype][0], kv_dtype, D)
    per = caches["bf16"][0].shape[0] // gc.B
    for b in range(gc.B):
        for i in range(pages):
            n = min(128, ids.shape[1] - 128 * i)
            want = mx.quantize(caches["bf16"][0][b * per + i, :, :, :n], kv_dtype)
            assert torch.equal(code[b * per + i, :, :, :n], want[0]) and torch.equal(scale[b * per + i, :, :, :n], want[1])
    # every row of the draft cache is a row of the block-scaled one
    values = mx.dequantize(code, scale, kv_dtype)
    kept = caches[kv_dtype][1]
    for half in (0, 1):
        for b in range(gc.B):
            dper = kept.shape[0] // gc.B
            rows = kept[b * dper:(b + 1) * dper, half].reshape(-1, *kept.shape[3:])[:gc.BUDGET].double()
            have = values[b * per:b * per + pages, half].transpose(1, 2).reshape(-1, *kept.shape[3:])[:ids.shape[1]]
            for h in range(kept.shape[3]):
                assert bool((torch.cdist(rows[:, h], have[:, h], compute_mode="donot_use_mm_for_euclid_dist").amin(1) == 0).all())
    assert torch.equal(logits[(kv_dtype, False)], logits[(kv_dtype, True)])
    assert torch.equal(outs[(kv_dtype, False)].output.cpu(), outs[(kv_dtype, True)].output.cpu())
    assert quantized_step_error(logits[(kv_dtype, False)], logits[("bf16", False)]) <= (2.0 ** -4 if kv_dtype == "mxfp8" else 0.25)


def test_select_in_groups_of_requests_is_the_select_of_all(ckpt_dir, monkeypatch):
    from magicdec_amd.Engine import model_core
    ids = next(iter(gc.synthetic_batches())).to(DEV)
    drafts = []
    for most in (model_core.MX_SELECT_BYTES, 1):
        monkeypatch.setattr(model_core, "MX_SELECT_BYTES", most)
        eng = engine(ckpt_dir, "mxfp8")
        eng.encode(ids)
        drafts.append([b.attention.kv_cache.draft_cache.clone() for b in eng.model.layers])
    for a, b in zip(*drafts):
        assert torch.equal(a, b)


def test_target_and_streaming_engines_run_on_block_scaled_pages(ckpt_dir):
    """The target of a speculation of two models, and the StreamingLLM self-speculation's verify cache."""
    from magicdec_amd.Engine.StreamingLLM.backend import LMBackend as Streaming
    ids = next(iter(gc.synthetic_batches())).to(DEV)
    tokens = {}
    for name, make in (("target", lambda kv: engine(ckpt_dir, kv, draft=False)), ("streaming", lambda kv: engine_streaming(ckpt_dir, kv, Streaming))):
        for kv in ("bf16", "mxfp8"):
            eng = make(kv)
            eng.encode(ids)
            (eng.inference if name == "target" else eng.verify)(ids[:, :gc.GAMMA + 1].clone())
            tokens[name, kv] = eng.model._last_logits.float().cpu()
        assert quantized_step_error(tokens[name, "mxfp8"], tokens[name, "bf16"]) <= 2.0 ** -4
        assert not torch.equal(tokens[name, "mxfp8"], tokens[name, "bf16"])


def engine_streaming(ckpt_dir, kv_dtype, cls):
    eng = cls(dtype=BF, device=DEV, dec_len=gc.GAMMA + 1)
    eng.load_model(os.path.join(ckpt_dir, "tinytgt", "model.pth"), use_tp=False)
    eng.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, draft_budget=gc.BUDGET, kv_dtype=kv_dtype)
    return eng


def test_other_layouts_and_caches_are_refused(ckpt_dir):
    from magicdec_amd.Engine.StreamingLLM.backend_draft import LMBackend_Draft
    with pytest.raises(ValueError, match="HND"):
        engine(ckpt_dir, "mxfp4", kv_layout="NHD")
    with pytest.raises(ValueError, match="kv_dtype"):
        engine(ckpt_dir, "mxfp6")
    assert "kv_dtype" not in LMBackend_Draft.setup_caches.__code__.co_varnames         # the ring cache is 16-bit
