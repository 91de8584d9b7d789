"""Cached decode with 8-bit projections."""
import pytest
import torch

import fp8_oracle as orc

pytestmark = pytest.mark.gpu

LAYERS = 4


def _model():
    from cverl_b200.models.config import Qwen35TextConfig
    from cverl_b200.models.qwen3_5 import Qwen35Model
    cfg = Qwen35TextConfig(vocab_size=2048, hidden_size=256, num_hidden_layers=LAYERS, num_attention_heads=4,
                           num_key_value_heads=2, head_dim=256, intermediate_size=512, linear_key_head_dim=128,
                           linear_value_head_dim=128, linear_num_key_heads=2, linear_num_value_heads=4)
    model = Qwen35Model(cfg, dtype=torch.bfloat16, device=torch.device("cuda", 0), with_main_grad=False)
    model.init_weights(seed=9)
    return model


def _steps(model, ids, fp8, graphed=False):
    from cverl_b200 import _native as nv
    from cverl_b200.models import decode
    with torch.no_grad():
        state, _ = decode.prefill(model, ids[:, :64], max_len=70)
        state.fp8 = fp8
        if graphed:
            runner = decode.GraphedDecoder(model, state, ids.shape[0], fp8=fp8)
            out = [runner.step(ids[:, t]).clone() for t in range(64, 70)]
        else:
            out = [decode.decode_step(model, state, ids[:, t]) for t in range(64, 70)]
    nv.check_status()
    assert state.length == 70
    return out


def _ids(batch):
    return torch.randint(1, 2048, (batch, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))


@pytest.mark.parametrize("batch", [1, 3, 130])
def test_decode_steps(batch, monkeypatch):
    """The kernels' steps, eager and from a graph, against the same steps with every 8-bit operator in 64 bits."""
    from cverl_b200 import ops
    from cverl_b200.models import decode
    model, ids = _model(), _ids(batch)
    weights = decode.fp8_decode_weights(model)
    eager, graph = _steps(model, ids, weights), _steps(model, ids, weights, graphed=True)
    for a, b in zip(eager, graph):
        assert torch.equal(a, b)

    def linear(x, w):
        x = x if isinstance(x, torch.Tensor) and x.dtype == torch.float64 else orc.through(x)
        return (x @ orc.value(w.w).t()).to(torch.bfloat16)

    def norm(x, r, w, eps, off):
        y, h, _ = orc.norm(x, r, w, eps, off)
        return orc.through(y), h

    monkeypatch.setattr(ops, "linear_fp8", linear)
    monkeypatch.setattr(ops, "add_rmsnorm_fp8", norm)
    # The two differ by fp32 sums, which move a value across a border of bf16 or of 8 bits now and then: less than the
    # bf16 rounding of every value, whose effect on this model is held to 4e-2 (the bf16 steps against fp32).
    for a, b in zip(eager, _steps(model, ids, weights)):
        assert (a - b).norm() <= 4e-2 * b.norm()


def test_every_projection_reads_its_own_weight(monkeypatch):
    """With the 8-bit operators replaced by the bf16 ones on the weight that was converted, the steps are the bf16 steps."""
    from cverl_b200 import ops
    from cverl_b200.models import decode
    model, ids = _model(), _ids(3)
    source = {}
    convert = ops.quantize_fp8_weight

    def remember(w, transposed=True):
        q = convert(w, transposed)
        source[id(q)] = (w, q)
        return q

    monkeypatch.setattr(ops, "quantize_fp8_weight", remember)
    weights = decode.fp8_decode_weights(model)
    assert len(weights) == 4 * LAYERS
    monkeypatch.setattr(ops, "linear_fp8", lambda x, w: ops.linear(x, source[id(w)][0]))
    monkeypatch.setattr(ops, "add_rmsnorm_fp8", ops.add_rmsnorm)
    for a, b in zip(_steps(model, ids, weights), _steps(model, ids, None)):
        assert torch.equal(a, b)


def test_weights_are_converted_anew_for_every_generation():
    from cverl_b200.rollout.worker import CachedQwenRolloutWorker, GenerationConfig, TokenBatch
    model = _model()
    worker = CachedQwenRolloutWorker(model, fp8=True)
    ids = torch.randint(1, 2048, (2, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    batch = TokenBatch(ids, torch.ones_like(ids), torch.full((2,), 64, device="cuda"))
    cfg = GenerationConfig(max_new_tokens=8, temperature=0.0, eos_token_id=-1, seed=0)
    first = worker.generate(batch, cfg)
    again = worker.generate(batch, cfg)
    assert torch.equal(first.token_ids, again.token_ids)
    model.init_weights(seed=10)
    assert not torch.equal(worker.generate(batch, cfg).token_ids, first.token_ids)


def test_models_without_the_native_step_are_refused():
    from cverl_b200.models import decode
    from cverl_b200.models.config import Qwen35TextConfig
    from cverl_b200.models.qwen3_5 import Qwen35Model
    model = Qwen35Model(Qwen35TextConfig.tiny(), dtype=torch.bfloat16, device=torch.device("cuda", 0), with_main_grad=False)
    with pytest.raises(RuntimeError, match="native decode"):
        decode.fp8_decode_weights(model)


def test_a_captured_decoder_keeps_its_weights():
    """The graph reads the weights that it was captured with, also after the state has been given others."""
    from cverl_b200.models import decode
    model, ids = _model(), _ids(2)
    want = _steps(model, ids, decode.fp8_decode_weights(model), graphed=True)
    with torch.no_grad():
        state, _ = decode.prefill(model, ids[:, :64], max_len=70)
        runner = decode.GraphedDecoder(model, state, 2, fp8=decode.fp8_decode_weights(model))
        sizes = [w.w.buf.numel() for w in state.fp8.values()]
        state.fp8 = None
        waste = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes]     # what freed memory would become
        got = [runner.step(ids[:, t]).clone() for t in range(64, 70)]
    del waste
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_which_policy_the_log_probs_come_from():
    """The first from the prompt's pass on the bf16 weights, the others from 8-bit steps over the caches it left."""
    from cverl_b200.models import decode
    from cverl_b200.rollout.worker import CachedQwenRolloutWorker, GenerationConfig, TokenBatch, sample_next_tokens
    model, ids = _model(), _ids(3)[:, :64].contiguous()
    batch = TokenBatch(ids, torch.ones_like(ids), torch.full((3,), 64, device="cuda"))
    cfg = GenerationConfig(max_new_tokens=3, temperature=0.0, eos_token_id=-1, seed=0)
    eight, sixteen = (CachedQwenRolloutWorker(model, fp8=f).generate(batch, cfg) for f in (True, False))
    assert torch.equal(eight.logprobs[:, 0], sixteen.logprobs[:, 0])
    assert not torch.equal(eight.logprobs[:, 1], sixteen.logprobs[:, 1])
    with torch.no_grad():
        state, logits = decode.prefill(model, ids, max_len=67)
        state.fp8 = decode.fp8_decode_weights(model)
        for t in range(3):
            tok, lp = sample_next_tokens(logits, cfg, None)
            assert torch.equal(eight.token_ids[:, t], tok) and torch.equal(eight.logprobs[:, t], lp)
            logits = decode.decode_step(model, state, tok)
