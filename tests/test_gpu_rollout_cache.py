"""The rollout engine with an 8-bit KV cache against the oracle's decode step over a cache that is quantised the same way: prompt
tokens attend unquantised rows, generated ones the quantised values.  The oracle is fed the engine's own tokens, so that the last step's logits
can be compared whatever a near-tie decided before; the tolerance is the one of the bf16 engine (test_gpu_rollout.py), since the
quantised values are the same on both sides (the oracle rounds them to bf16 once more, 2^-9 of a value)."""
import numpy as np
import pytest
import torch

from oracle import decode as dec
from oracle.rollout import QwenConfig, decode_step, rope_tables, seeded_params
from pcp_b200 import BackendError
from pcp_b200 import backend as bk
from pcp_b200.backend import Rollout

SMALL = QwenConfig(vocab=1024, d_model=512, n_layer=2, n_head=4, n_kv_head=2, head_dim=128, d_ff=1024, max_seq=64, dtype="bf16")
HD64 = QwenConfig(vocab=1000, d_model=512, n_layer=1, n_head=8, n_kv_head=2, head_dim=64, d_ff=512, max_seq=48, dtype="bf16")


def _engine(cfg, cache, **kw):
    return Rollout(0, cfg.vocab, cfg.d_model, cfg.n_layer, cfg.n_head, cfg.n_kv_head, cfg.head_dim, cfg.d_ff, cfg.max_seq, max_batch=kw.get("max_batch", 6),
                   max_prompt=cfg.max_seq, page_tokens=4, rope_theta=cfg.rope_theta, rms_eps=cfg.rms_eps, cache=cache)


def _quantised(row, kind):
    return dec.values(*dec.quantise(row, kind)).to(torch.bfloat16)


def _oracle_last_logits(cfg, params, prompt, tokens, kind):
    params = [p.to(cfg.torch_dtype) for p in params]
    tables = rope_tables(cfg)
    kc, vc = ([torch.zeros(cfg.n_kv_head, cfg.max_seq, cfg.head_dim, dtype=cfg.torch_dtype) for _ in range(cfg.n_layer)] for _ in range(2))
    prompt = prompt or [0]
    for pos, tok in enumerate(prompt + tokens[:-1]):
        if pos == len(prompt):                                   # the prompt is done: what it wrote is read as codes from here on
            for l in range(cfg.n_layer):
                for c in (kc, vc):
                    c[l][:, :pos] = _quantised(c[l][:, :pos], kind)
        logits, kn, vn = decode_step(cfg, params, tok, pos, kc, vc, tables)
        for l in range(cfg.n_layer):
            kc[l][:, pos] = kn[l] if pos < len(prompt) else _quantised(kn[l], kind)
            vc[l][:, pos] = vn[l] if pos < len(prompt) else _quantised(vn[l], kind)
    return logits.float().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["e4m3", "i8"])
@pytest.mark.parametrize("cfg", [SMALL, HD64], ids=["hd128", "hd64"])
def test_decode_over_a_quantised_cache(cfg, kind):
    params = seeded_params(cfg, seed=0, std=0.05, head_std=1.0)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab, size=n).tolist() for n in (9, 1, 17, 5, 12)] + [[]]
    blob = np.concatenate([p.to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16).reshape(-1) for p in params])
    with _engine(cfg, kind) as eng, _engine(cfg, "bf16") as plain:
        for e in (eng, plain):
            e.ensure_device_weights(blob)
        first, _, _ = eng.generate_rollout(prompts, 1)
        assert first == plain.generate_rollout(prompts, 1)[0]    # the prompt pass does not see the codes
        for new in (2, 5):
            got, why, _ = eng.generate_rollout(prompts, new)
            assert why == ["length"] * len(prompts)
            for b, p in enumerate(prompts):
                ref = _oracle_last_logits(cfg, params, p, got[b], kind)
                have = eng.read_logits(b)
                assert np.abs(have - ref).max() <= 2e-2 * np.abs(ref).max(), (new, b)
        assert eng.generate_rollout(prompts, 5)[0] == got        # pages and the captured step are used again
        assert eng.generate_rollout(prompts[:2], 5)[0] == got[:2]          # another batch, another graph


def test_cache_types():
    with pytest.raises(ValueError):
        _engine(SMALL, "f16")
    if not torch.cuda.is_available():
        with pytest.raises(BackendError) as ei:
            _engine(SMALL, "i8")
        assert ei.value.code == bk.E_CUDA
