"""The decoder of bench_decoder.py with its queries and keys rotated, cached and attended to by the library's operators: against the same decode step
through torch's operations, and one layer's attention over codes against the codes read back."""
import pytest
import torch

pytestmark = pytest.mark.gpu

bd = pytest.importorskip("bench_decoder")


def rel(a, b):
    return ((a.float() - b.float()).abs().max() / b.float().abs().max().clamp_min(1e-6)).item()


@pytest.fixture(scope="module")
def model():
    from bitween_amd import Bitween
    with torch.device("cuda"):
        m = bd.Decoder(layers=2, hidden=512, heads=4, inter=1024, vocab=1000, max_len=96).half()
    m.init_weights(seed=3)
    m = Bitween(m, bits=4, group_size=128).quantize(rtn=True, ignore_layers=["lm_head", "embed_tokens"], verbose=False)
    m.alloc_state()
    return m


@pytest.fixture
def ids():
    return torch.randint(0, 1000, (40,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))


# The bar is the one of the decoder's other glue: float16 roundings of every torch operation against one rounding of an operator.
@pytest.mark.parametrize("glue", [False, True])
def test_16_bits_are_the_decoder_s_own_step(model, ids, glue):
    model.paged = model.glue = None
    model.prefill(ids)
    want = model.step().clone()
    kv = model.kv.clone()
    model.use_paged_cache(16, page_size=32)
    if glue:
        model.use_hip_glue(splits=4)
    model.kv.zero_()
    model.prefill(ids)
    assert rel(model.step(), want) < 1e-2
    slots = model.paged[0].slots(model.page_table, torch.arange(41, device="cuda"), torch.zeros(41, dtype=torch.int64, device="cuda"))
    for i, cache in enumerate(model.paged):
        for got, layer_kv in zip(cache.read(slots), kv[i]):
            assert rel(got.transpose(0, 1), layer_kv[0, :, :41]) < 1e-2
    assert not model.kv.any()


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 32)])
def test_a_captured_step_generates_the_same_tokens(model, ids, bits, group):
    model.glue = None
    model.use_paged_cache(bits, group, page_size=16)
    _, _, eager = bd.generate(model, ids, 24)
    graph = bd.capture_step(model)
    for _ in range(3):
        _, _, tokens = bd.generate(model, ids, 24, graph)
        assert torch.equal(tokens, eager)


# Reading back rounds keys and values to float16 (2^-11), which moves a score by at most 2^-11 sum |q k| / sqrt(128) < 2^-11 * 16 = 2^-7 here and an output by
# that, 2^-11 of its own and of the values: below 1e-2 of the largest.
@pytest.mark.parametrize("bits,group", [(8, 64), (8, 128), (4, 32)])
def test_attention_over_codes_is_that_over_the_values_read_back(model, bits, group):
    model.use_paged_cache(bits, group, page_size=16)
    gen = torch.Generator(device="cuda").manual_seed(bits + group)
    q, k, v = (torch.randn(60, 512, device="cuda", generator=gen).half() for _ in range(3))
    pos = torch.arange(60, device="cuda")
    model._place(pos)
    rotated, _, _ = model._rotate_and_cache(1, q, k, v, pos)
    keys, values = (x.double().transpose(0, 1) for x in model.paged[1].read(model._slots))
    assert 128 ** -0.5 * (rotated[-1].double()[:, None].abs() * keys.abs()).sum(-1).max() < 16
    scores = (rotated[-1].double()[:, None] * keys).sum(-1) * 128 ** -0.5
    want = (scores.softmax(-1)[..., None] * values).sum(1)
    model.pos.fill_(59)
    model._place(model.pos)
    assert rel(model._attend_paged(q[-1:], k[-1:], v[-1:], 1).view(4, 128), want) < 1e-2
