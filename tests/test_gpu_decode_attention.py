"""A decode step that attends: projections, cache append and paged attention run together as a model runs them."""
import pytest
import torch

import lowlat_gemm as L
from lowlat_gemm import _native as N, tp as TP

from test_gpu_attention import BF, E4M3, HF, plain_quantised

pytestmark = pytest.mark.gpu

SHAPE = TP.LayerShape(hidden=1024, qkv=1536, inter=2048)  # 8 query heads, 2 kv heads of 128


def recorded(step):
    """The step's gemm calls as (layer projection, input, output), in order."""
    calls, inner = [], step._gemm

    def gemm(x, w, **kw):
        y = inner(x, w, **kw)
        calls.append((x.clone(), y.clone()))
        return y

    step._gemm = gemm
    return calls


@pytest.mark.parametrize("kind,dtype", [("bf16", E4M3), ("bf16", BF), ("f16", HF), ("f16", E4M3), ("w8a16_bf16", E4M3)])
@pytest.mark.parametrize("new", [1, 3])
def test_step_attends_to_everything_before(kind, dtype, new):
    batch, layers, steps, dev = 3, 2, 4, torch.device("cuda", 0)
    cache = TP.DecodeCache(layers, batch, 64, 2, dev, page_size=16, dtype=dtype)
    step = TP.DecodeStep(kind, layers, 1, 0, dev, SHAPE, residual=True, cache=cache)
    act = step.act_dtype
    calls = recorded(step)
    keys = [[[] for _ in range(batch)] for _ in range(layers)]
    values = [[[] for _ in range(batch)] for _ in range(layers)]
    half = torch.finfo(act).eps / 2
    g = torch.Generator().manual_seed(5)
    for t in range(steps):
        calls.clear()
        x = (torch.randn(batch * new, 1024, generator=g) * 0.5).to(act).to(dev)
        step.run(x)
        assert len(calls) == 4 * layers and cache.kv_lens.tolist() == [(t + 1) * new] * batch
        for li in range(layers):
            qkv, attn = calls[4 * li][1], calls[4 * li + 1][0]
            q, k, v = (z.view(batch * new, -1, 128) for z in qkv.split([1024, 256, 256], dim=1))
            for i in range(batch):
                for j in range(new):
                    for rows, store in ((k, keys), (v, values)):
                        row = rows[i * new + j]
                        if dtype == E4M3:
                            val, e = plain_quantised(row)
                            row = torch.ldexp(val.double(), e[:, None])
                        store[li][i].append(row.double())
                kk, vv = torch.stack(keys[li][i]), torch.stack(values[li][i])
                for j in range(new):
                    n = kk.shape[0] - new + j + 1
                    for h in range(8):
                        s = kk[:n, h // 4] @ q[i * new + j, h].double() / 128 ** 0.5
                        p = torch.softmax(s, 0)
                        want = p @ vv[:n, h // 4]
                        mass = p @ vv[:n, h // 4].abs()
                        # one rounding of the result and one of each probability; a score is off by (128 + 4) * 2^-24 of its
                        # sum of magnitudes and moves a weight by twice that
                        delta = (kk[:n, h // 4].abs() @ q[i * new + j, h].double().abs()).max() / 128 ** 0.5 * 132 * 2.0 ** -24 + 2.0 ** -20
                        got = attn[i * new + j, h * 128:(h + 1) * 128].double()
                        assert bool(((got - want).abs() <= half * want.abs() + mass * (half + 2 * delta) + torch.finfo(act).tiny).all())
    assert N.device_status() == 0


def test_captured_step_appends_on_every_replay():
    batch, dev = 2, torch.device("cuda", 0)
    x = (torch.randn(batch, 1024, generator=torch.Generator().manual_seed(1)) * 0.5).to(BF).to(dev)

    def fresh():
        cache = TP.DecodeCache(1, batch, 100, 2, dev, page_size=16)
        return cache, TP.DecodeStep("fp8", 1, 1, 0, dev, SHAPE, residual=True, cache=cache)

    cache, step = fresh()
    want = [step.run(x).clone() for _ in range(6)]
    cache2, step2 = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step2.run(x)
    torch.cuda.current_stream().wait_stream(side)
    cache2.kv_lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step2.run(x)
    cache2.kv_lens.zero_()
    for w in want:
        graph.replay()
        assert torch.equal(y, w)
    assert cache2.kv_lens.tolist() == [6, 6] and torch.equal(cache.layers[0][0][0].view(torch.uint8), cache2.layers[0][0][0].view(torch.uint8))


def test_without_a_cache_the_step_is_what_it_was():
    dev = torch.device("cuda", 0)
    x = (torch.randn(4, 1024, generator=torch.Generator().manual_seed(2)) * 0.5).to(BF).to(dev)
    step = TP.DecodeStep("bf16", 1, 1, 0, dev, SHAPE)
    calls = recorded(step)
    step.run(x)
    assert torch.equal(calls[1][0], calls[0][1][:, :1024])


def test_refusals():
    dev = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="kv heads"):
        TP.DecodeStep("bf16", 1, 1, 0, dev, SHAPE, cache=TP.DecodeCache(1, 2, 64, 4, dev))
    with pytest.raises(ValueError, match="kv heads"):
        TP.DecodeStep("bf16", 2, 1, 0, dev, SHAPE, cache=TP.DecodeCache(1, 2, 64, 2, dev))
    with pytest.raises(ValueError, match="do not split"):
        TP.DecodeStep("bf16", 1, 1, 0, dev, TP.LayerShape(hidden=1024, qkv=1024, inter=2048), cache=TP.DecodeCache(1, 2, 64, 2, dev))
    step = TP.DecodeStep("bf16", 1, 1, 0, dev, SHAPE, cache=TP.DecodeCache(1, 2, 64, 2, dev))
    with pytest.raises(ValueError, match="no multiple"):
        step.run(torch.zeros(3, 1024, dtype=BF, device=dev))
