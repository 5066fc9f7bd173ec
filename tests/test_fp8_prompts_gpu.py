"""GPU: prompts of a Qwen2 in 8 bits, and what does not run in 8 bits."""
import pytest
import torch

from tests.test_fp8_gpu import nothing_left_behind, qwen, rand  # noqa: F401
from tests.test_fp8_prompts_cpu import in_turn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("S", [1, 40, 300])
def test_constrained_decoding_is_bf16_behind_an_8_bit_prompt(cuda, S):
    """Each step's logits are the bf16 model's from the same cache, bit by bit."""
    llm, emb, toks = qwen().prefill_in_fp8(), rand(3, S, 512).to(BF).to(cuda), [3, 500, 7, 999]
    seen, choose = [], in_turn(*toks)

    def processor(hist, scores):
        seen.append(scores[0].clone())
        return choose(hist, scores)

    ids = llm.generate(inputs_embeds=emb[None], max_new_tokens=4, eos_token_id=None, logits_processor=[processor])
    assert ids.tolist() == [toks]
    cache = llm.new_cache(S + 4)
    hid = llm.prefill_hidden(emb, cache)
    llm.prefill_in_fp8(False)
    for i, tok in enumerate(toks):
        assert torch.equal(llm.logits_from_hidden(hid[-1:])[0].float(), seen[i])
        hid = llm.prefill_hidden(llm.model.embed_tokens(torch.tensor([tok], device=cuda)), cache)


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_weights_made_by_generate_are_made_anew_by_forward(cuda, mode):
    llm, emb = qwen(layers=2).prefill_in_fp8(), rand(4, 90, 512).to(BF).to(cuda)
    llm.generate(inputs_embeds=emb[None], max_new_tokens=2, eos_token_id=None)      # in inference mode
    with torch.no_grad():
        llm.model.layers[1].mlp.down_proj.weight.mul_(2)
    with mode():
        got = llm.forward(inputs_embeds=emb[None]).logits
    assert torch.equal(llm.forward(inputs_embeds=emb[None]).logits, got)
    other = qwen(layers=2)
    with torch.no_grad():
        other.model.layers[1].mlp.down_proj.weight.mul_(2)
    assert torch.equal(other.prefill_in_fp8().forward(inputs_embeds=emb[None]).logits, got)
