"""MXFP4SelfAttention's cache: the prompt's weights, evictions, captured steps."""

import pytest
import torch

from .test_gpu_kv_cache import formula, held, reference_evict
from .test_gpu_operators import layer_of

pytestmark = pytest.mark.gpu


def prompt_weights(layer, x, lens, cache, page, dev):
    """In 64 bits: the weight of each held key over its prompt's queries, and the
    bound on its error."""
    from lockstep_amd import fp4
    from lockstep_amd.mxfp4_gemm import mxfp4_linear_w
    q = layer._split(mxfp4_linear_w(x, *layer.packed[0]))[0]
    at = 0
    for b, n in enumerate(lens):
        if n:
            kc, ks, _, _ = held(cache.pages, cache.table, b, n, page, dev)
            k = fp4.dequantize_packed(kc.contiguous().flatten(0, 1), ks.contiguous().flatten(0, 1)).view(n, *kc.shape[1:2], -1)
            _, _, w, err = formula(q[at:at + n], k, k, layer.window, layer.sinks, layer.head_dim ** -0.5)
            yield b, n, w, err
        at += n


@pytest.mark.parametrize("rows", [16384, 128])     # in one pass, in several
@pytest.mark.parametrize("window,sinks,lens", [(None, 2, [70, 0, 30, 200]), (40, 3, [300, 129]), (None, 0, [1])])
def test_prefill_accumulates_the_prompts_weights(window, sinks, lens, rows, dev, monkeypatch):
    from lockstep_amd import fp4_attention
    monkeypatch.setattr(fp4_attention, "_WEIGHT_ROWS", rows, raising=False)
    layer = layer_of(dev, window=window, sinks=sinks).pack()
    for longest in (max(lens), None):
        cache = layer.new_cache(len(lens), 512, page_size=16, track=True)
        x = torch.randn((sum(lens), 512), generator=torch.Generator(device=dev).manual_seed(3), device=dev).bfloat16()
        offsets = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=dev)
        layer.prefill(x, cache, offsets, longest=longest)
        for b, n, w, err in prompt_weights(layer, x, lens, cache, 16, dev):
            bad = (cache.weights[b, :, :n].double() - w).abs() - err - 2.0 ** -20 * w
            assert bad.max().item() <= 0, (b, bad.max().item())
        for b, n in enumerate(lens):
            assert (cache.weights[b, :, n:] == 0).all()


def test_eviction_straight_after_a_prompt(dev):
    """What stays is what the prompt attended to: every token has a weight, its own at least."""
    layer = layer_of(dev, sinks=1).pack()
    cache = layer.new_cache(2, 256, page_size=16, track=True)
    x = torch.randn((300, 512), generator=torch.Generator(device=dev).manual_seed(5), device=dev).bfloat16()
    layer.prefill(x, cache, torch.tensor([0, 200, 300], dtype=torch.int32, device=dev), longest=200)
    w = cache.weights.cpu()
    index = cache.evict(64, recent=8)
    for b, n in enumerate((200, 100)):
        for h in range(2):
            assert index[b, h].tolist() == reference_evict(w[b, h].tolist(), n, 64, 1, 8)
            assert (w[b, h, :n] > 0).all()


def test_captured_steps_go_on_after_an_eviction(dev):
    """A captured step replays on what eager calls, evictions and other replays left."""
    layer = layer_of(dev, window=50, sinks=2).pack()
    g = torch.Generator(device=dev).manual_seed(9)
    prompts = torch.randn((100, 512), generator=g, device=dev).bfloat16()
    offsets = torch.tensor([0, 60, 100], dtype=torch.int32, device=dev)
    caches = [layer.new_cache(2, 128, page_size=16, track=True) for _ in range(2)]
    x = torch.randn((2, 1, 512), generator=g, device=dev).bfloat16()
    for c in caches:
        layer.prefill(prompts, c, offsets, longest=60)
        layer.step(x, c)
    eager, captured = caches
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, eager)
    torch.cuda.current_stream().wait_stream(side)
    layer.step(x, captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(x, captured)      # recorded, not run: its token is counted by the host alone
    captured.used -= 1
    for i in range(40):
        x.copy_(torch.randn((2, 1, 512), generator=g, device=dev))
        want = layer.step(x, eager)
        captured.reserve(1)
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(captured.lengths, eager.lengths) and captured.used == eager.used
        assert torch.equal(captured.weights, eager.weights)
        if i % 13 == 12:
            assert torch.equal(captured.evict(40, recent=6), eager.evict(40, recent=6))


def test_a_prompt_of_no_sequence(dev):
    layer = layer_of(dev).pack()
    x = torch.randn((7, 512), generator=torch.Generator(device=dev).manual_seed(2), device=dev).bfloat16()
    cache = layer.new_cache(0, 40, page_size=16, track=True)
    assert (layer.prefill(x, cache, torch.zeros(1, dtype=torch.int32, device=dev)) == 0).all()
    assert cache.weights.shape == (0, 2, 48)
