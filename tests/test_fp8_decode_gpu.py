"""Cached decode with 8-bit projections."""
import pytest
import torch

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


@pytest.mark.parametrize("batch", [1, 3, 130])
def test_decode_steps(batch):
    from cverl_b200 import _native as nv
    from cverl_b200.models import decode
    model = _model()
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(1, 2048, (batch, 70), device="cuda", generator=g)
    weights = decode.fp8_decode_weights(model)
    runs = {}
    with torch.no_grad():
        for name, fp8, graphed in (("bf16", None, False), ("eager", weights, False), ("graph", weights, True)):
            state, _ = decode.prefill(model, ids[:, :64], max_len=70)
            if graphed:
                runner = decode.GraphedDecoder(model, state, batch, fp8=fp8)
                runs[name] = [runner.step(ids[:, t]).clone() for t in range(64, 70)]
            else:
                state.fp8 = fp8
                runs[name] = [decode.decode_step(model, state, ids[:, t]) for t in range(64, 70)]
            assert state.length == 70
    nv.check_status()
    for a, b in zip(runs["eager"], runs["graph"]):
        assert torch.equal(a, b)
    # a rounding to e4m3 is at most 2^-4 of a value; a block has two products of two rounded operands each, a layer two
    # blocks, and the roundings do not know of each other: the root of their number
    for a, b in zip(runs["eager"], runs["bf16"]):
        assert (a - b).norm() <= 2.0 ** -4 * (4 * 2 * LAYERS) ** 0.5 * b.norm()
        assert not torch.equal(a, b)


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
