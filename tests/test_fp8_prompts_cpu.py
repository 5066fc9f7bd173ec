"""CPU: which of a Qwen2's steps run in 8 bits, with the kernels stood in for."""
import pytest
import torch

from vila_b200 import ops
from vila_b200.model import qwen2
from vila_b200.model.configuration import Qwen2Config


def in_turn(*ids):
    """A logits processor that has these tokens chosen one after another."""
    left = list(ids)

    def choose(hist, scores):
        scores = torch.full_like(scores, -1e4)
        scores[:, left.pop(0)] = 0
        return scores
    return choose


@pytest.fixture
def llm(monkeypatch):
    """A model whose operators give random rows of the right shapes; calls: (operator, rows) of every layer that it asks for."""
    cfg = Qwen2Config(hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=50)
    m = qwen2.Qwen2ForCausalLM(cfg, device="cpu")
    with torch.no_grad():
        for p in m.state_dict().values():
            p.normal_()
    m.calls = []

    def rows(name, n=None):
        def run(x, w, *a, swiglu=False, out=None, to8=False, **k):
            m.calls.append((name, x.shape[0]))
            width = w.shape[0] // 2 if swiglu else w.shape[0]
            if to8:
                return ops.Fp8._alloc(w._held(), x.shape[0], width, 1)
            return out if out is not None else torch.randn(x.shape[0], width).bfloat16()
        return run

    def norm8(x, w, eps, residual=None, out=None):
        return ops.Fp8._alloc(x, *x.shape, 1), x if out is None else out

    fakes = dict(linear=rows("bf16"), fp8_linear=rows("fp8"), fp8_rmsnorm=norm8, rmsnorm=lambda x, w, eps: x, linear_qkv_rope=lambda *a, **k: None,
                 rope_table=lambda *a: None, rope_kv_append=lambda *a: None, rope_kv_append_table=lambda *a: None, fmha=lambda q, *a, **k: q.clone(),
                 gemv=lambda x, w, **k: torch.randn(w.shape[0]).bfloat16(), check_waits=lambda: None,
                 fp8_quantize=lambda w, block_rows=1: m.calls.append(("quantise", w.shape[0])) or ops.Fp8._alloc(w, *w.shape, block_rows))
    for name, fake in fakes.items():
        monkeypatch.setattr(ops, name, fake)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(qwen2.Embedding, "forward", lambda self, ids: self.weight.detach()[ids])
    return m


@pytest.mark.parametrize("how", ["processor", "sampled"])
def test_sampled_and_constrained_decoding_stays_bf16(llm, how):
    llm.prefill_in_fp8()
    emb = torch.randn(7, 64).bfloat16()
    more = dict(logits_processor=[in_turn(3, 5, 2, 4)]) if how == "processor" else dict(do_sample=True)
    ids = llm.generate(inputs_embeds=emb[None], max_new_tokens=4, eos_token_id=None, **more)
    assert ids.shape == (1, 4)
    eight, plain = [n for name, n in llm.calls if name == "fp8"], [n for name, n in llm.calls if name == "bf16"]
    assert eight == [7] * 8                       # the prompt: four projections a layer
    assert plain == [1] * 8 * 4                   # every decoded token


@pytest.mark.parametrize("first, then", [("inference", "plain"), ("inference", "no_grad"), ("plain", "inference"), ("inference", "inference")])
def test_8_bit_weights_follow_a_change_in_either_mode(llm, first, then):
    """Weights made at a prompt in inference mode are made anew, in the same memory, at one outside of it, and the other way round."""
    modes = dict(inference=torch.inference_mode, plain=torch.enable_grad, no_grad=torch.no_grad)
    llm.prefill_in_fp8()
    emb = torch.randn(3, 64).bfloat16()

    def prompt(mode):
        del llm.calls[:]
        with modes[mode]():
            llm.forward(inputs_embeds=emb[None])
        return [name for name, _ in llm.calls].count("quantise"), [q for qs in llm._fp8_weights() for q in qs]

    made, held = prompt(first)
    assert made == 8 and not any(q._held().is_inference() for q in held)
    assert prompt(first)[0] == prompt(then)[0] == 0
    with torch.no_grad():
        llm.model.layers[1].mlp.down_proj.weight.mul_(2)
    made, again = prompt(then)
    assert made == 8 and [q._held().data_ptr() for q in again] == [q._held().data_ptr() for q in held]
    assert prompt(then)[0] == prompt(first)[0] == 0
    assert prompt(first)[0] == 0 and llm.prefill_in_fp8() is llm and prompt(then)[0] == 8
