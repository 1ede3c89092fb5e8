"""Index arrays and scales off their 4-byte boundaries are refused on the host by the operators over grouped rows: the kernels
read them as words."""
from __future__ import annotations

import pytest

from test_cpu_grouped_rows import MISALIGNED, P, build, combine, combine_grad, dw, gather, lora, mm, route


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call,args", [
    (build, dict(ids=P)), (build, dict(offsets=P)), (build, dict(order=P)), (build, dict(pos=P)),
    (gather, dict(pos=P)), (combine, dict(pos=P)), (combine_grad, dict(pos=P)),
    (mm, dict(offsets=P)), (dw, dict(offsets=P)), (lambda **k: mm(fn="spmm_grouped_mm_dx", **k), dict(offsets=P)),
    (lora, dict(offsets=P)), (lora, dict(adapter=P)), (lora, dict(scale=P)),
    (lambda **k: lora(rank=0, **k), dict(scale=P)),  # read even where there is nothing to scale
])
def test_words_off_their_boundaries(call, args, off):
    (name, at), = args.items()
    if name == "pos" and call is not build:
        assert call(r=route(pos=at + off)) == MISALIGNED
    else:
        assert call(**{name: at + off}) == MISALIGNED
