"""``generate`` with rules on its logits and with 4-bit projections: the whole chain against the same steps taken one by one."""
import pytest
import torch

import hf_adapter_b200 as hb

pytestmark = pytest.mark.gpu
V = 300


def model_of(fmt=None, dtype=torch.float16):
    torch.manual_seed(4)
    cfg = hb.NativeRWKV7Config(vocab_size=V, hidden_size=256, num_hidden_layers=2, num_heads=4, head_dim=64, intermediate_size=512,
                               decay_low_rank_dim=32, a_low_rank_dim=32, v_low_rank_dim=16, gate_low_rank_dim=32)
    model = hb.RWKV7ForCausalLM(cfg)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(0.2 * torch.randn_like(p) if p.dim() < 2 else torch.randn_like(p) * p.shape[-1] ** -0.5)
        model.lm_head.weight.mul_(4)
    model = model.to(dtype).cuda().eval()
    if fmt:
        hb.quantize_model(model, fmt, min_params=1, skip=())
    return model


def step_by_step(model, ids, n, pick):
    """The loop of ``generate`` with ``pick(logits, ids so far)`` for a token."""
    out = model(ids, logits_to_keep=1)
    cache, logits = out.past_key_values, out.logits[:, -1]
    for step in range(n):
        if step:
            logits = model.rwkv7_forward_token(tok, cache)
        tok = pick(logits, ids)
        ids = torch.cat((ids, tok[:, None]), 1)
    return ids


@pytest.mark.parametrize("fmt", [None, "nvfp4", "mxfp4"])
@pytest.mark.parametrize("do_sample", [False, True])
def test_penalties_bias_and_draw(fmt, do_sample):
    model = model_of(fmt)
    ids = torch.randint(0, V, (3, 6), device="cuda")
    bias = torch.zeros(V, device="cuda")
    bias[5], bias[7] = 2.0, -float("inf")
    presence = torch.tensor([0.5, 0.0, 1.0], device="cuda")
    gen = lambda: torch.Generator(device="cuda").manual_seed(9)
    more = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01) if do_sample else {}
    got = model.generate(ids, max_new_tokens=8, do_sample=do_sample, generator=gen(), repetition_penalty=1.3, presence_penalty=presence,
                         frequency_penalty=0.2, logit_bias=bias, **more)
    g = gen()

    def pick(logits, so_far):
        z = logits.float()
        for b in range(3):  # the rules, a row at a time
            seen = so_far[b].unique()
            z[b, seen] = torch.where(z[b, seen] > 0, z[b, seen] / 1.3, z[b, seen] * 1.3)
            c = torch.bincount(so_far[b, 6:], minlength=V).float()
            z[b] = z[b] - 0.2 * c - presence[b] * (c > 0)
        z = z + bias
        if not do_sample:
            return z.argmax(-1)
        noise = torch.empty(3, V, device="cuda").exponential_(generator=g)
        return hb.sample_tokens(z, noise, **more)

    assert torch.equal(got, step_by_step(model, ids, 8, pick))
    assert not (got[:, 6:] == 7).any()


def test_penalties_skip_padding():
    """A padded prompt is penalised for its tokens, not for its padding: the same continuation as without padding."""
    model = model_of(dtype=torch.float32)
    ids = torch.randint(1, V, (1, 5), device="cuda")
    padded = torch.cat((torch.zeros(1, 3, device="cuda", dtype=ids.dtype), ids), 1)
    mask = torch.cat((torch.zeros(1, 3, device="cuda", dtype=ids.dtype), torch.ones_like(ids)), 1)
    a = model.generate(ids, max_new_tokens=6, repetition_penalty=5.0)
    b = model.generate(padded, attention_mask=mask, max_new_tokens=6, repetition_penalty=5.0)
    assert torch.equal(a[:, 5:], b[:, 8:])
    new = a[0, 5:].tolist()
    assert len(set(new)) == len(new)  # (a penalty of 5 lets nothing come back here)


def test_grammar_masks():
    model = model_of("nvfp4")
    ids = torch.randint(0, V, (2, 4), device="cuda")

    def words(rows):
        m = torch.zeros(2, (V + 31) // 32 * 32, dtype=torch.int64, device="cuda")
        for b, r in enumerate(rows):
            m[b, list(r)] = 1
        w = (m.view(2, -1, 32) << torch.arange(32, device="cuda")).sum(-1)
        return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()

    calls = []

    def grammar(new):
        calls.append(new.clone())
        return words([{10 + new.shape[1], 31}, {299} if new.shape[1] < 2 else set()])

    out = model.generate(ids, max_new_tokens=5, allowed_tokens=grammar, pad_token_id=3)
    assert [int(c.shape[1]) for c in calls] == [0, 1, 2, 3, 4]
    assert all(int(out[0, 4 + t]) in (10 + t, 31) for t in range(5))
    assert out[1, 4:].tolist() == [299, 299, 3, 3, 3]  # row 1 may say nothing more from its third token on
    fixed = model.generate(ids, max_new_tokens=3, allowed_tokens=words([{8}, {9}]), do_sample=True)
    assert fixed[:, 4:].tolist() == [[8] * 3, [9] * 3]
    assert model.generate(ids, max_new_tokens=5, allowed_tokens=words([set(), set()]), pad_token_id=1).tolist() == [r + [1] for r in ids.tolist()]
