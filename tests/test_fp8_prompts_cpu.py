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


def test_only_weights_that_were_waited_for_are_fetched_ahead(llm, monkeypatch):
    """A layer asks for its weight ahead of what the launch before wrote only where the weight says so: those of a model behind a synchronisation."""
    from types import SimpleNamespace
    weight = ops.Fp8(torch.zeros(64, 64).to(torch.float8_e4m3fn), torch.ones(1, 1), 128)
    kept = ops.Fp8Kept(ops.Fp8(torch.zeros(64, 64).to(torch.float8_e4m3fn), torch.ones(1, 1), 128), torch.zeros(8, 64).bfloat16())
    x, asked = torch.zeros(3, 64).bfloat16(), []
    monkeypatch.undo()
    monkeypatch.setattr(ops, "_mx4_here", lambda t, name: None)
    monkeypatch.setattr(ops, "_chk", lambda t, name: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    lib = SimpleNamespace(vila_fp8_linear_scratch=lambda p: 0, vila_fp8_linear=lambda p, stream: asked.append(p._obj.flags & 2) or 0)
    monkeypatch.setattr(ops._lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "linear", lambda x, w, bias, static_w, out: asked.append(2 * static_w))
    for call in (lambda: ops.fp8_linear(x, weight), lambda: ops.linear_any(x, weight)):
        weight.static_w = False
        call()
        weight.static_w = True
        call()
    assert asked == [0, 2, 0, 2]
    ops.linear_any(x, kept)
    kept.static_w = True
    ops.linear_any(x, kept)
    assert asked[4:] == [0, 0, 2, 2]
    assert not ops.Fp8._alloc(x, 4, 64, 128).static_w and not ops.Fp8(weight.codes, weight.scales, 128).static_w


def test_a_prompts_weights_are_fetched_ahead_once_they_were_waited_for(llm, monkeypatch):
    waited, made = [], []
    quantise = ops.fp8_quantize
    monkeypatch.setattr(ops, "fp8_quantize", lambda w, block_rows: made.append(quantise(w, block_rows=block_rows)) or made[-1])
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: waited.append((len(made), any(q.static_w for q in made))))
    eights = llm.prefill_in_fp8()._fp8_weights()
    assert waited == [(0, False), (8, False)] and all(q.static_w for qs in eights for q in qs)


@pytest.mark.parametrize("weights, asked, told", [(None, 0, False), ("fp8", 1, False), ("mx4", 0, True)])
def test_weights_of_a_vision_language_checkpoint(monkeypatch, tmp_path, capsys, weights, asked, told):
    """fp8 runs its prompts in 8 bits; mx4, which it never had, is accepted as it always was, and says that it does nothing."""
    import warnings
    from types import SimpleNamespace
    from llava.cli import infer
    calls = []
    fake = SimpleNamespace(llm=SimpleNamespace(prefill_in_fp8=lambda: calls.append("fp8")), config=SimpleNamespace(),
                           generate_content=lambda prompt, response_format=None: "an answer")
    monkeypatch.setattr(infer.llava, "load", lambda path, model_base=None: fake)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        got = infer.main(["--model-path", str(tmp_path), "--text", "hello"] + (["--weights", weights] if weights else []))
    assert got == "an answer" and "an answer" in capsys.readouterr().out
    assert calls == ["fp8"] * asked and any("token-id language models" in str(w.message) for w in seen) == told


def test_weights_are_copied_whole():
    import copy
    part = ops.Fp8(torch.zeros(64, 64).to(torch.float8_e4m3fn), torch.ones(1, 1), 128)
    for w in (part, ops.Fp8Kept(part, torch.zeros(8, 64).bfloat16())):
        w.static_w = True
        for other in (copy.deepcopy(w), copy.copy(w)):
            assert type(other) is type(w) and other.shape == w.shape and other.static_w
            assert torch.equal(getattr(other, "part", other).codes.float(), part.codes.float())
