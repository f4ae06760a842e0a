"""The ctypes registration of the paged-cache operators: another process, where it is the one in use, computes the same bits."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import lowlat_gemm as L

from test_gpu_attention import BF, E4M3, make_cache, pages_for

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def chain(ct):
    """Append, both attention kernels, with offsets and without, and read; on fixed inputs."""
    lens, out = [70, 300, 33], []
    table, pages = pages_for(lens, 16, 1)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 128, ct, 2)
    scales = dict(k_scale=ks, v_scale=vs)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(3)
    for new, starts in ((1, None), (30, None), (1, [0, 1, 2, 3]), (30, [0, 60, 61, 90])):
        kv = torch.randn(3 * new, 4, 128, generator=g).to(BF).cuda()
        q = torch.randn(3 * new, 8, 128, generator=g).to(BF).cuda()
        st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
        L.kv_append(kv[:, :2], kv[:, 2:], kc, vc, table, ln, q_starts=st, **scales)
        out += L.paged_attention(q, kc, vc, table, ln, q_starts=st, window=50, return_lse=True, **scales)
    out += L.kv_read(kc, vc, table, ln, 300, **scales)
    return [t.cpu() for t in out]


REFUSALS = '''
import pytest, torch, lowlat_gemm as L
from lowlat_gemm import _native as N, _ops
assert _ops.BACKEND == "ctypes"
kc = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
table, ln = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
q = torch.zeros(3, 8, 128, dtype=torch.bfloat16, device="cuda")
for text, fn, args, kw in (
        ("must have q's type", L.paged_attention, (q.half(), kc, kc, table, ln), {}),
        ("1 to 32 times", L.paged_attention, (q[:, :7], kc, kc, table, ln), {}),
        ("window", L.paged_attention, (q, kc, kc, table, ln), dict(window=-1)),
        ("must be on", L.paged_attention, (q, kc, kc, table.cpu(), ln), {}),
        ("k_scale is needed", L.paged_attention, (q, kc.to(torch.float8_e4m3fn), kc.to(torch.float8_e4m3fn), table, ln), {}),
        ("the cache holds", L.kv_append, (q, q, kc, kc, table, ln), {}),
        ("16-bit cache's type", L.kv_read, (kc, kc, table, ln, 4), dict(out_dtype=torch.float16))):
    with pytest.raises(RuntimeError, match=text):
        fn(*args, **kw)
assert N.device_status() == 0
'''


def test_the_ctypes_registration_gives_the_same_bits(tmp_path):
    code = f"import sys; sys.path[:0] = [{str(ROOT / 'sm120-lowlat-gemm_b200')!r}, {str(ROOT / 'tests')!r}]\n{REFUSALS}\n" \
        f"import test_gpu_attention_ctypes as T\ntorch.save([T.chain(T.BF), T.chain(T.E4M3)], {str(tmp_path / 'out.pt')!r})\n"
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, LLG_OPS="ctypes"), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    for got, ct in zip(torch.load(tmp_path / "out.pt"), (BF, E4M3)):
        want = chain(ct)
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
