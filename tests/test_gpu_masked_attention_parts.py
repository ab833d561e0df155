"""Masked attention's dK / dV where a key block's steps are shared by a cluster of eight."""
import math
import random

import pytest
import torch

from tests.support import packed_reference as ref
from tests.test_gpu_masked_attention import inputs, make_ids, mask_of, run

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


# key blocks whose steps a cluster of eight shares (on 148 SMs): few key blocks, many query heads to each
@pytest.mark.parametrize("B,S,Hk,G,kind,softcap,bias,token_major", [(1, 65, 1, 8, "one", 0.0, False, True), (1, 300, 1, 14, "prefix", 0.0, False, False),
                                                                    (1, 300, 1, 8, "docs", 20.0, True, True), (2, 130, 1, 9, "docs", 0.0, False, True)])
def test_key_blocks_shared_by_eight(cuda_device, B, S, Hk, G, kind, softcap, bias, token_major):
    ids, prefix = make_ids(kind, B, S, S + G)
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, 64, BF16, token_major, S)
    slopes = 2.0 ** -torch.arange(1, Hk * G + 1, device=cuda_device, dtype=F32) if bias else None
    want = ref.attention(q, k, v, dout, ids, prefix, G, 0.125, softcap, slopes, token_major, BF16, True)
    mask = mask_of(cuda_device, ids, prefix)
    got = run(q, k, v, dout, G, 0.125, mask, softcap, slopes, token_major)
    for name, value in want.items():
        ref.check(got[name], value, name)
    again = run(q, k, v, dout, G, 0.125, mask, softcap, slopes, token_major)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("bad", [None, math.nan, math.inf])
def test_eight_parts_of_which_some_are_empty(cuda_device, bad):
    """Two query heads over documents of up to 70 of 4096 positions: a key block has two to six steps for its eight parts.  With values that are
    not finite in every other document, key rows beside them are taken again."""
    S, G, d, rng = 4096, 2, 64, random.Random(2)
    ids, spans = [], []
    while len(ids) < S:
        n = min(S - len(ids), rng.randint(1, 70))
        spans.append((len(ids), len(ids) + n))
        ids += [len(spans) % 5] * n
    q, k, v, dout = inputs(cuda_device, 1, S, 1, G, d, BF16, False, 9)
    base = [t.clone() for t in (q, k, v, dout)]
    if bad is not None:
        for a, e in spans[::2]:
            for t, n in ((q, G), (k, 1), (v, 1), (dout, G)):
                t.view(n, S, d)[:, a:e] = bad
    got = run(q, k, v, dout, G, 0.125, mask_of(cuda_device, [ids], None), 0.0, None, False)
    for a, e in spans[1::2]:
        part = lambda t, n: t.view(n, S, -1)[:, a:e].reshape(1, n * (e - a), -1).contiguous()  # noqa: E731
        want = ref.attention(part(base[0], G), part(base[1], 1), part(base[2], 1), part(base[3], G), [[0] * (e - a)], None, G, 0.125, 0.0, None, False, BF16, True)
        for name, n in (("o", G), ("dq", G), ("dk", 1), ("dv", 1)):
            ref.check(part(got[name], n), want[name], f"{name} of [{a}, {e})")
