"""The operators of a windowed decoder together, as bench_decoder.py runs them: a prompt through rotation, cache write and prompt_attention, then one token at a time through
append and attention over the pages."""
import pytest
import torch

from prompt_ref import visible

pytestmark = pytest.mark.gpu

bd = pytest.importorskip("bench_decoder")
WINDOW, SINKS, PROMPT, STEPS = 24, 3, 40, 17


def _rel(a, b):
    return ((a.double() - b).abs().max() / b.abs().max()).item()


@pytest.fixture(scope="module")
def model():
    from bitween_amd import Bitween
    with torch.device("cuda"):
        m = bd.Decoder(layers=2, hidden=512, heads=4, inter=1024, vocab=1000, max_len=96).half()
    m.init_weights(seed=3)
    m = Bitween(m, bits=4, group_size=128).quantize(rtn=True, ignore_layers=["lm_head", "embed_tokens"], verbose=False)
    m.alloc_state()
    return m


# 16 bits: the kernels round weights (2^-11, and 2^-9 of dot products in scores below 16 in float32 is nothing) and outputs once, the cache nothing: 2^-9 of the largest is four times that.
# 8 and 4 bits: the reference takes what the cache gives back (rounded once more to float16, 2^-11 of keys and values, scores below 16: 2^-7); the prompt's attention takes what came in.
@pytest.mark.parametrize("bits,group,page", [(16, 0, 32), (8, 64, 16), (4, 32, 16)])
@pytest.mark.parametrize("seed", [0, 1])
def test_a_prompt_and_steps_see_the_window(model, bits, group, page, seed):
    from bitween_amd import rotate_heads
    model.glue = None
    model.use_paged_cache(bits, group, page_size=page, window=WINDOW, sinks=SINKS)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = PROMPT + STEPS
    q, k, v = (torch.randn(total, 512, device="cuda", generator=gen).half() for _ in range(3))
    at = torch.arange(total, device="cuda")
    heads = [x.view(total, 4, 128) for x in (q, k, v)]
    turned, keys = rotate_heads(heads[0], heads[1], model.cos32, model.sin32, at)
    model._place(at[:PROMPT])
    got = [model._attend_prompt(*model._rotate_and_cache(1, q[:PROMPT], k[:PROMPT], v[:PROMPT], at[:PROMPT]))]
    for t in range(PROMPT, total):
        model.pos.fill_(t)
        model._place(model.pos)
        got.append(model._attend_paged(q[t:t + 1], k[t:t + 1], v[t:t + 1], 1).view(1, 4, 128))
    got = torch.cat(got)
    slots = model.paged[1].slots(model.page_table, at, torch.zeros_like(at))
    kept = [x.double() for x in model.paged[1].read(slots)]
    if bits == 16:
        assert torch.equal(kept[0], keys.double()) and torch.equal(kept[1], heads[2].double())
    seen = visible(total, total, WINDOW, SINKS)
    for part, (kk, vv) in ((slice(0, PROMPT), (keys.double(), heads[2].double())), (slice(PROMPT, total), kept)):
        scores = torch.matmul(turned.double().transpose(0, 1), kk.permute(1, 2, 0)) * 128 ** -0.5
        assert scores.abs().max() < 16
        want = torch.matmul(scores.masked_fill(~seen, float("-inf")).softmax(-1), vv.transpose(0, 1)).transpose(0, 1)
        assert _rel(got[part], want[part]) < (2.0 ** -9 if bits == 16 or part.start == 0 else 1e-2)


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64)])
@pytest.mark.parametrize("glue", [False, True])
def test_a_captured_step_generates_the_same_tokens(model, bits, group, glue):
    ids = torch.randint(0, 1000, (PROMPT,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    model.glue = None
    model.use_paged_cache(bits, group, page_size=16, window=WINDOW, sinks=SINKS)
    if glue:
        model.use_hip_glue(splits=4)
    _, _, eager = bd.generate(model, ids, 24)
    graph = bd.capture_step(model)
    for _ in range(3):
        _, _, tokens = bd.generate(model, ids, 24, graph)
        assert torch.equal(tokens, eager)


def test_a_step_appends_what_rotation_and_cache_write_leave(model):
    """Bit for bit: one kernel in place of two."""
    model.glue = None
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(1, 512, device="cuda", generator=gen).half() for _ in range(3))
    for bits, group in ((16, 0), (8, 64), (4, 32)):
        rows, outs = [], []
        for one in (True, False):
            model.use_paged_cache(bits, group, page_size=16)
            model.pos.fill_(33)
            model._place(model.pos)
            if one:
                outs.append(model._attend_paged(q, k, v, 0).view(1, 4, 128))
            else:
                turned, _, _ = model._rotate_and_cache(0, q, k, v, model.pos)
                outs.append(model.paged[0].attend(turned, model.page_table, model._lengths))
            rows.append(model.paged[0].read(model._slots))
        assert torch.equal(*outs) and all(torch.equal(a, b) for a, b in zip(*rows))
