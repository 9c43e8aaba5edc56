"""The step metadata of the hybrid decoder (StepMeta) on the host: the running totals of the sequences' positions are kept
for caches in 4 bits alone, and a step without them fills as many words as its fields have."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

HOST = SimpleNamespace(int32=torch.int32, zeros=lambda n, dtype, **kw: torch.full((n,), -7, dtype=dtype))


def meta(**kw):
    from exl3_b200.hybrid import StepMeta

    return StepMeta(HOST, "cpu", 12, 4, 3, **kw)


def fill(m, rows_of):
    offs = np.concatenate([[0], np.cumsum([n for _, n in rows_of])]).astype(int)
    seq = [s for s, (_, n) in enumerate(rows_of) for _ in range(n)]
    pos = [p + i for p, n in rows_of for i in range(n)]
    m.fill(range(len(pos)), seq, pos, offs, [3 - s for s in range(len(rows_of))], [0])
    return offs


STEPS = [[(0, 5)], [(7, 1), (0, 3)], [(7, 1), (9, 1), (0, 1)], [(4, 0), (2, 2), (30, 0)], [(1, 1)]]


@pytest.mark.parametrize("rows_of", STEPS)
def test_contexts_of_a_step(rows_of):
    m = meta(contexts=True)
    fill(m, rows_of)
    want = np.concatenate([[0], np.cumsum([p + n if n else 0 for p, n in rows_of])])
    o = m.off["kv_offsets"]
    assert m.host[o:o + len(want)].tolist() == want.tolist() and m.kv_total == want[-1]
    assert m.len["kv_offsets"] == 5 and m.host.numel() == o + 5


@pytest.mark.parametrize("rows_of", STEPS)
def test_steps_without_contexts_have_none(rows_of):
    m = meta()
    n = 3 * 12 + 2 * 4 + 1 + 3
    assert m.host.numel() == m.dev.numel() == n and "kv_offsets" not in m.off
    offs = fill(m, rows_of)
    assert m.host[m.off["row_offsets"]:][:len(offs)].tolist() == offs.tolist()
    assert m.kv_total == 0 and m.one_row_each == all(k == 1 for _, k in rows_of)


def test_no_rows():
    for contexts in (False, True):
        m = meta(contexts=contexts)
        m.fill([], [], [], [0], [], [])
        assert m.kv_total == 0 and not m.one_row_each
