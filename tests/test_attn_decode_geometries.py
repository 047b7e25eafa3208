"""Which int8-KV head sizes decode attention serves and which it refuses: 64 over a
slice of a wider cache, against the CPU oracle, and sizes that no kernel is built for."""

import pytest
import torch

from oracle import attention as A
from test_attn_decode import DEV, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 2)])
def test_head_64_over_the_first_half_of_wider_caches(strix, hq, hkv):
    lens, bs, hd = [40, 1, 300, 0], 16, 64
    q, kc, vc, _, seq_lens, table = A.build_paged_kv([1] * len(lens), lens, hq, hkv, bs, hd=hd)
    (kq, ks), (vq, vs) = A.quantize_kv(kc), A.quantize_kv(vc)
    ref = A.decode_reference(q, kq, vq, ks, vs, seq_lens, table, hd ** -0.5)
    wide = [torch.full((*t.shape[:3], 128), 127, dtype=torch.int8, device=DEV) for t in (kq, vq)]
    wide[0][..., :hd], wide[1][..., :hd] = kq.to(DEV), vq.to(DEV)
    out = torch.full_like(q, float("nan"), device=DEV)
    strix.attn_decode(out, q.to(DEV), wide[0][..., :hd], wide[1][..., :hd], seq_lens.to(DEV), table.to(DEV),
                      hd ** -0.5, 1, -1, ks.to(DEV), vs.to(DEV))
    check(out, ref)


@pytest.mark.parametrize("hd", [32, 96, 120])
def test_other_head_sizes_are_refused(strix, hd):
    q = torch.zeros(1, 8, hd, dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(4, 16, 8, hd, dtype=torch.int8, device=DEV)
    scale = torch.ones(4, 16, 8, device=DEV)
    meta = torch.ones(1, dtype=torch.int32, device=DEV), torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="not built"):
        strix.attn_decode(torch.empty_like(q), q, cache, cache, *meta, 0.1, 1, -1, scale, scale)
