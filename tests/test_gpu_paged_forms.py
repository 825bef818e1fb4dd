"""Every form of the paged-cache kernels (the calls of paged_forms.py) against float64."""

from __future__ import annotations

import numpy as np
import paged_forms as forms
import paged_ref as ref
import pytest

torch = pytest.importorskip("torch")

from rtxllm_amd import paged  # noqa: E402
from test_gpu_paged import DEV, Setup, close, dev, u32  # noqa: E402

pytestmark = pytest.mark.gpu


def calls(table):
    return [pytest.param(form, c, id=f"{form}-{c}") for form, cs in table.items() for c in cs]


@pytest.mark.parametrize("form,shape", calls(forms.APPEND))
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
def test_append(form, shape, pairing):
    heads, kv, dim, count = shape
    s = Setup(heads + dim, [count], kv, dim, 16, one=True)
    rng = s.rng
    q, k, v = (rng.standard_normal((count, h, dim)).astype(np.float32) for h in (heads, kv, kv))
    w = (1.0 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    pos = rng.permutation(count).astype(np.uint32)
    pad = rng.random(count) < 0.05
    rotary = dim if pairing == "halves" else dim // 2
    out = torch.full((count, heads, dim), 7.0, device=DEV)
    paged.qk_norm_rope_append(s.cache, dev(q), dev(k), dev(v), dev(w), None, u32(np.where(pad, ref.NONE, pos)), theta=1e5,
                              rotary_dim=rotary, pairing=pairing, q_out=out)
    gk, gv, got = s.kd.cpu().numpy(), s.vd.cpu().numpy(), out.cpu().numpy()
    i = np.arange(rotary // 2)
    a, b = (i, i + rotary // 2) if pairing == "halves" else (2 * i, 2 * i + 1)
    angle = pos[:, None].astype(np.float64) * 1e5 ** (-2.0 * i / rotary)
    c, sn = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def form_of(x, weight):
        y = x.astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * weight
        z, size = y.copy(), np.abs(y)
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * sn, y[..., a] * sn + y[..., b] * c
        size[..., a] = size[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
        return z, size

    # fp32, as in test_gpu_paged.test_append: 24 roundings from the sum of squares to the rotation
    live = ~pad
    want, size = form_of(q, w.astype(np.float64))
    close(got[live], want[live], 24 * 2.0 ** -24 * size[live], "q")
    assert np.all(got[pad] == 7.0)
    want, size = form_of(k, 1.0)
    p, o = np.array(s.seen[0])[pos[live]].T
    close(gk[p, :, o], want[live], 2.0 ** -11 * np.abs(want[live]) + 48 * 2.0 ** -24 * size[live] + 2.0 ** -25, "k")
    k_want, v_want = s.k.copy(), s.v.copy()
    k_want[p, :, o], v_want[p, :, o] = gk[p, :, o], v[live].astype(np.float16)
    np.testing.assert_array_equal(gk.view(np.uint16), k_want.view(np.uint16))
    np.testing.assert_array_equal(gv.view(np.uint16), v_want.view(np.uint16))


@pytest.mark.parametrize("form,shape", calls(forms.BOUNDS))
def test_page_bounds(form, shape):
    kv, dim, page, filled, span = shape
    s = Setup(dim + page + span, list(filled), kv, dim, page)
    want = s.rng.standard_normal((s.n_pages, kv, 2, dim)).astype(np.float16)
    bounds = dev(want)
    paged.page_bounds(s.cache, u32(s.last()), bounds, None if span == 1 else u32([0] * len(filled)), span)
    for i, n in enumerate(filled):
        used = -(-n // page)
        for t in range(used - 1 if span == 1 and n else 0, min(span, used) if span > 1 else used):
            p = s.table[i, t]
            for g in range(kv):
                want[p, g] = ref.bounds_of(s.k[p, g, :min(page, n - t * page)])
    np.testing.assert_array_equal(bounds.cpu().numpy(), want)


@pytest.mark.parametrize("form,shape", calls(forms.SCORE))
def test_select_pages(form, shape):
    group, kv, dim, filled = shape
    s = Setup(group + dim, list(filled), kv, dim, 1)
    bounds = np.sort(s.rng.standard_normal((s.n_pages, kv, 2, dim)).astype(np.float16), axis=2)[:, :, ::-1]
    q = s.rng.standard_normal((len(filled), group * kv, dim)).astype(np.float32)
    scores = {}
    for i, n in enumerate(filled):
        for g in range(kv):
            x, b = q[i, g * group:(g + 1) * group].astype(np.float64), bounds[s.table[i, :n], g].astype(np.float64)
            scores[i, g] = (np.maximum(x, 0.0) @ b[:, 0].T + np.minimum(x, 0.0) @ b[:, 1].T).max(0)
    bd, qd = dev(bounds), dev(q)
    for first, last, select in ((0, 0, 37), (1, 2, 900)):
        pages = torch.full((len(filled), kv, select), -9, dtype=torch.int32, device=DEV)
        paged.select_pages(s.cache, bd, qd, u32(s.last()), select, first, last, pages=pages)
        got = pages.cpu().numpy()
        for (i, g), score in scores.items():
            n = filled[i]
            if n == 0:
                assert np.all(got[i] == -9)
                continue
            score = score.copy()
            score[:first], score[max(0, n - last):] = np.inf, np.inf
            order = np.argsort(-score, kind="stable")[:select]
            assert got[i, g].tolist() == sorted(order.tolist()) + [-1] * (select - len(order)), (i, g)


@pytest.mark.parametrize("form,shape", calls(forms.EVICT))
@pytest.mark.parametrize("place", ["apart", "in-place"])
def test_evict(form, shape, place):
    count, kv, dim, page, slots, keep = shape
    lens = [slots] * count
    lens[1] = keep  # nothing leaves
    s = Setup(dim + page + keep, lens, kv, dim, page)
    rng = s.rng
    weight = (rng.integers(0, 40, (count, kv, s.capacity)) / 8).astype(np.float32)
    weight[:, :, ::9] = np.nan
    slot_pos = np.stack([[rng.permutation(s.capacity) for _ in range(kv)] for _ in range(count)]).astype(np.uint32)
    newest = [int(p[:, :n].max()) for p, n in zip(slot_pos, lens)]
    if count > 3:
        newest[3] = ref.NONE  # a padded row
    wd, sd, ld = dev(weight), u32(slot_pos), u32(lens)
    apart = place == "apart"
    outs = [torch.full_like(t, 7) for t in (wd, sd, ld)] if apart else [wd, sd, ld]
    paged.evict(s.cache, ld, u32(newest), keep, wd, sd, 2, 15, *(outs if apart else ()))
    gw, gp, gl = outs[0].cpu().numpy(), outs[1].cpu().numpy().view(np.uint32), outs[2].cpu().tolist()
    k_want, v_want = s.k.copy(), s.v.copy()
    for i, n in enumerate(lens):
        if newest[i] == ref.NONE:
            assert gl[i] == (7 if apart else n)
            continue
        assert gl[i] == min(n, keep)
        at = np.array(s.seen[i])
        for g in range(kv):
            src = ref.evict(n, newest[i], keep, 2, 15, weight[i, g], slot_pos[i, g])
            src = np.arange(n) if src is None else np.array(src)
            np.testing.assert_array_equal(gw[i, g, :len(src)], weight[i, g, src])
            np.testing.assert_array_equal(gp[i, g, :len(src)], slot_pos[i, g, src])
            to = np.flatnonzero(src != np.arange(len(src)))
            (p, o), (p2, o2) = at[to].T, at[src[to]].T
            k_want[p, g, o], v_want[p, g, o] = s.k[p2, g, o2], s.v[p2, g, o2]
    np.testing.assert_array_equal(s.kd.cpu().numpy().view(np.uint16), k_want.view(np.uint16))
    np.testing.assert_array_equal(s.vd.cpu().numpy().view(np.uint16), v_want.view(np.uint16))
