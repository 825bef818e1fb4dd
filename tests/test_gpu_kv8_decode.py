"""The 8-bit cache and the attention of new rows as a serving program uses them together: a prompt, then
tokens one at a time, eagerly and as a captured step; workspaces, streams, repeats, sizes past 32 bits and past a launch's
dimensions; what the wrappers refuse."""

from __future__ import annotations

import numpy as np
import pytest
import rows_ref as ref

torch = pytest.importorskip("torch")

from rtxllm_amd import kv8, paged  # noqa: E402
from rtxllm_amd._lib import HipError, lib  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPE = dict(int8=torch.int8, e4m3=torch.float8_e4m3fn)


def dev(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def u32(values) -> torch.Tensor:
    return dev(np.asarray(values, np.uint32).view(np.int32))


class Serving:
    """Sequences with prompts in an 8-bit cache; q, k and v of every position to come."""

    def __init__(self, seed, fmt, lens, steps, kv=2, group=4, dim=128, page=64, block=16):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.steps, self.kv, self.group, self.dim = lens, steps, kv, group, dim
        entries = -(-(max(lens) + steps) // page)
        n_pages = entries * len(lens) + 1
        self.table = rng.permutation(n_pages)[:entries * len(lens)].astype(np.int32).reshape(len(lens), -1)
        self.args = (n_pages, kv, page, dim, block)
        self.fmt, self.m = fmt, ref.Model(self.table, n_pages, kv, page, dim, block, fmt)
        most = max(lens) + steps
        self.x = [rng.standard_normal((len(lens), most, kv, dim)).astype(np.float32) for _ in range(2)]
        self.q = rng.standard_normal((len(lens), most, kv * group, dim)).astype(np.float32)

    def cache(self):
        return kv8.PagedKV8.empty(*self.args, dev(self.table), DTYPE[self.fmt])

    def prompt(self, cache, window, sinks):
        parts = [np.concatenate([x[i, :n] for i, n in enumerate(self.lens)]) for x in (self.x[0], self.x[1], self.q)]
        start = u32(np.cumsum([0] + self.lens))
        kv8.append(cache, dev(parts[0]), dev(parts[1]), u32([0] * len(self.lens)), start)
        return kv8.attn(cache, dev(parts[2]), u32([0] * len(self.lens)), start, window=window, sinks=sinks)

    def token(self, i):
        """(k, v, q) of each sequence's i-th token behind its prompt."""
        return [np.stack([x[s, n + i] for s, n in enumerate(self.lens)]) for x in (self.x[0], self.x[1], self.q)]

    def check(self, out, i, window, sinks):
        """The step's results against float64, from the model that took the same tokens."""
        got = out.cpu().numpy()
        for s, n in enumerate(self.lens):
            p = n + i
            j = ref.visible(p, window, sinks)
            for g in range(self.kv):
                keys, values = (np.stack([self.m.value(c, s, g, int(t), p + 1) for t in j]) for c in range(2))
                for h in range(g * self.group, (g + 1) * self.group):
                    want, tol = ref.attend(self.q[s, p, h], keys, values)
                    assert bool((np.abs(got[s, h] - want) <= tol).all()), (s, i, h)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(1 << 24, 0), (48, 4)])
def test_prompt_then_tokens(fmt, window, sinks):
    """Two caches: one steps eagerly, one by a captured step whose position grows on the device, with the first one's
    work between its replays. Both follow the float64 model, bit for bit alike."""
    s = Serving(1, fmt, [75, 33, 100], 22)
    eager, graphed = s.cache(), s.cache()
    a, b = s.prompt(eager, window, sinks), s.prompt(graphed, window, sinks)
    assert torch.equal(a, b)
    for i, n in enumerate(s.lens):
        s.m.append(i, 0, [x[i, :n] for x in s.x])
    rows = len(s.lens)
    pos, k, v, q = u32(s.lens), *(dev(x) for x in s.token(0))
    out = torch.zeros_like(q)
    work = kv8.attn_workspace(graphed, s.kv * s.group, rows, rows, window, sinks)
    spare = s.cache()

    def step(cache):
        kv8.append(cache, k, v, pos)
        kv8.attn(cache, q, pos, window=window, sinks=sinks, out=out, workspace=work)
        pos.add_(1)

    step(spare)  # (loads what a first call loads)
    pos.copy_(u32(s.lens))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(graphed)
    torch.cuda.synchronize()
    for i in range(s.steps):
        new = s.token(i)
        for t, x in zip((k, v, q), new):
            t.copy_(dev(x))
        graph.replay()
        at = u32([n + i for n in s.lens])
        kv8.append(eager, dev(new[0]), dev(new[1]), at)
        want = kv8.attn(eager, dev(new[2]), at, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for j in range(rows):
            s.m.append(j, s.lens[j] + i, [x[j:j + 1] for x in new[:2]])
        if i % 7 == 3:
            s.check(out, i, window, sinks)
    for x, y in ((eager.k, graphed.k), (eager.v, graphed.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_drafts_taken_back():
    """Drafts that are dropped: the next tokens go over them within the newest block, or from a block's start."""
    s = Serving(2, "int8", [45], 30)
    kept, tried = s.cache(), s.cache()
    for c in (kept, tried):
        s.prompt(c, 1 << 24, 0)
    wrong = [dev(s.rng.standard_normal((19, s.kv, s.dim)).astype(np.float32)) for _ in range(2)]
    kv8.append(tried, wrong[0][:3], wrong[1][:3], u32([45]), u32([0, 3]))  # 45..47 make a block whole
    kv8.append(tried, *(dev(x[0, 32:45]) for x in s.x), u32([32]), u32([0, 13]))  # back to the block's start
    kv8.append(tried, wrong[0][:2], wrong[1][:2], u32([45]), u32([0, 2]))
    for c in (kept, tried):
        kv8.append(c, *(dev(x[0, 45:52]) for x in s.x), u32([45]), u32([0, 7]))
    q = dev(s.q[0, 45:52])
    a, b = (kv8.attn(c, q, u32([45]), u32([0, 7])) for c in (kept, tried))
    assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["f16", "int8"])
@pytest.mark.parametrize("rows", ["tokens", "drafts", "prompt"])
def test_calls_repeat_whatever_the_workspace_holds(fmt, rows):
    """The same bits from a workspace of NaN and from one of another call; nothing is written behind it."""
    rng = np.random.default_rng(3)
    kv, group, dim, page, n = 2, 4, 128, 64, 3000
    entries = -(-n // page)
    table = dev(rng.permutation(entries).astype(np.int32).reshape(1, -1))
    if fmt == "f16":
        k, v = (torch.randn(entries, kv, page, dim, device=DEV).half() for _ in range(2))
        cache, space, run = paged.PagedKV(k, v, table), paged.attn_window_workspace, paged.attn_window
    else:
        cache = kv8.PagedKV8.empty(entries, kv, page, dim, 16, table)
        x = [torch.randn(n, kv, dim, device=DEV) for _ in range(2)]
        kv8.append(cache, *x, u32([0]), u32([0, n]))
        space, run = kv8.attn_workspace, kv8.attn
    new = dict(tokens=1, drafts=5, prompt=200)[rows]
    q = torch.randn(new, kv * group, dim, device=DEV)
    start = None if new == 1 else u32([0, new])
    need = space(cache, kv * group, 1, new).numel()
    work = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device=DEV)
    first = run(cache, q, u32([n - new]), start, workspace=work[:need])
    assert (work[need:] == 0xFF).all()
    again = run(cache, q, u32([n - new]), start, workspace=work[:need])
    assert torch.equal(first, again) and bool(first.isfinite().all())
    with pytest.raises(ValueError):
        run(cache, q, u32([n - new]), start, workspace=work[:need - 256])


def test_two_streams_and_two_graphs():
    """Two captured steps on streams of their own, with a workspace each, replayed together."""
    s = Serving(4, "int8", [2000, 700], 2)
    cache = s.cache()
    s.prompt(cache, 1 << 24, 0)
    q = [dev(s.rng.standard_normal((2, 8, 128)).astype(np.float32)) for _ in range(2)]
    pos = u32([n - 1 for n in s.lens])
    want = [kv8.attn(cache, x, pos) for x in q]
    out = [torch.zeros_like(x) for x in q]
    work = [kv8.attn_workspace(cache, 8, 2, 2) for _ in q]
    streams, graphs = [torch.cuda.Stream() for _ in q], [torch.cuda.CUDAGraph() for _ in q]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            with torch.cuda.graph(graphs[i], stream=streams[i]):
                kv8.attn(cache, q[i], pos, out=out[i], workspace=work[i])
    for _ in range(5):
        for x in out:
            x.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_one_token_of_very_many_sequences():
    """More units than one dimension of a launch holds."""
    count, kv, dim, page = 40000, 1, 64, 8
    table = torch.arange(count, dtype=torch.int32, device=DEV).reshape(-1, 1)
    cache = kv8.PagedKV8.empty(count, kv, page, dim, 8, table)
    x = [torch.randn(count, kv, dim, device=DEV).half().float() for _ in range(2)]
    zero = torch.zeros(count, dtype=torch.int32, device=DEV)
    kv8.append(cache, *x, zero)
    q = torch.randn(count, 2, dim, device=DEV)
    got = kv8.attn(cache, q, zero)
    assert torch.allclose(got, x[1].expand(count, 2, dim), rtol=2.0 ** -20, atol=0.0)  # one position: its value
    start = torch.arange(count + 1, dtype=torch.int32, device=DEV)
    assert torch.allclose(kv8.attn(cache, q, zero, start), got, rtol=2.0 ** -20, atol=0.0)


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_past_32_bit_offsets(fmt):
    """Pages behind 4 GiB of each cache: rows read there are those that were put there."""
    page, kv, dim = 1024, 8, 256
    n_pages = (1 << 32) // (page * kv * dim) + 3
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    n = 2 * page + 129
    x = [torch.randn(n, kv, dim, device=DEV, generator=g).half() for _ in range(2)]
    small = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    outs = []
    for t, pages in ((table, n_pages), (small, 3)):
        if fmt == "f16":
            k, v = (torch.zeros(pages, kv, page, dim, dtype=torch.float16, device=DEV) for _ in range(2))
            cache = paged.PagedKV(k, v, t)
            for i in range(3):
                part = [y[i * page:(i + 1) * page].transpose(0, 1) for y in x]
                p = int(t[0, i])
                k[p, :, :part[0].shape[1]], v[p, :, :part[1].shape[1]] = part[0], part[1]
            run = paged.attn_window
        else:
            cache = kv8.PagedKV8.empty(pages, kv, page, dim, 64, t)
            kv8.append(cache, *x, u32([0]), u32([0, n]))
            run = kv8.attn
        q = torch.randn(130, kv, dim, device=DEV, generator=g.manual_seed(7)).half()
        outs.append([run(cache, q[:1], u32([n - 1])), run(cache, q, u32([n - 130]), u32([0, 130]))])
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.isfinite().all())


def test_beside_the_listed_pages_of_the_fp16_cache():
    """Over fp16 pages without a window, one token a sequence is what attention over all pages, listed, gives."""
    rng = np.random.default_rng(8)
    kv, group, dim, page, lens = 4, 4, 128, 32, [500, 77, 1]
    entries = -(-500 // page)
    n_pages = entries * 3
    k, v = (dev(rng.standard_normal((n_pages, kv, page, dim)).astype(np.float16)) for _ in range(2))
    cache = paged.PagedKV(k, v, dev(rng.permutation(n_pages).astype(np.int32).reshape(3, -1)))
    q = dev(rng.standard_normal((3, kv * group, dim)).astype(np.float32))
    pos = u32([n - 1 for n in lens])
    pages = torch.arange(entries, dtype=torch.int32, device=DEV).expand(3, kv, entries).contiguous()
    a, b = paged.attn_window(cache, q, pos), paged.attn_pages(cache, q, pages, pos)
    assert bool((a - b).abs().max() <= 2.0 ** -16 * v.abs().max())  # both within their bounds of 500 positions' sums


def test_wrappers_refuse():
    s = Serving(9, "int8", [40], 4)
    c = s.cache()
    k, v = (torch.zeros(5, 2, 128, device=DEV) for _ in range(2))
    q = torch.zeros(5, 8, 128, device=DEV)
    one, start = u32([0]), u32([0, 5])
    bad = [lambda: kv8.append(c, k.double(), v, one, start), lambda: kv8.append(c, k, v.half(), one, start),
           lambda: kv8.append(c, k, v[:2], one, start), lambda: kv8.append(c, k, v, one), lambda: kv8.append(c, k.cpu(), v, one, start),
           lambda: kv8.append(c, k[..., ::2], v, one, start), lambda: kv8.append(c, k, v, one, u32([0, 1, 5])),
           lambda: kv8.append(c, k, v, u32([0, 0]), u32([0, 1, 5])), lambda: kv8.append(c, k, v, one.long(), start),
           lambda: kv8.read(c, one, one, start), lambda: kv8.read(c, one, one, dtype=torch.bfloat16),
           lambda: kv8.read(c, one, u32([0, 0])), lambda: kv8.read(c, one, one, k_out=torch.zeros(1, 2, 64, device=DEV)),
           lambda: kv8.attn(c, q.double(), one, start), lambda: kv8.attn(c, q[:, :7], one, start), lambda: kv8.attn(c, q, one),
           lambda: kv8.attn(c, q, one, start, window=-1), lambda: kv8.attn(c, q, one, start, window=0),
           lambda: kv8.attn(c, q, one, start, sinks=1 << 33), lambda: kv8.attn(c, q, one, start, out=q.half()),
           lambda: kv8.attn(c, q, one, start, workspace=torch.zeros(1 << 20, dtype=torch.uint8)),
           lambda: kv8.attn(c, q.view(5, 1024), one, start), lambda: kv8.attn_workspace(c, 7, 1, 5),
           lambda: kv8.PagedKV8(c.k.half(), c.v.half(), c.k_scale, c.v_scale, c.k_tail, c.v_tail, c.block_table),
           lambda: kv8.PagedKV8(c.k, c.v, c.k_scale[:, :, :1].contiguous(), c.v_scale, c.k_tail, c.v_tail, c.block_table),
           lambda: kv8.PagedKV8(c.k, c.v, c.k_scale, c.v_scale, c.k_tail[:, :, :12].contiguous(), c.v_tail, c.block_table),
           lambda: kv8.PagedKV8(c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, c.block_table[0]),
           lambda: kv8.PagedKV8(c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, c.block_table.expand(2, -1))]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, HipError)):
            f()
            pytest.fail(f"call {i} is not refused")
    with pytest.raises(HipError):  # (no rows: nothing to do is refused, as by the library)
        kv8.append(c, k[:0], v[:0], one, u32([0, 0]))
    over = torch.zeros(5 * 8 * 128 + 64, device=DEV)
    with pytest.raises(HipError):
        kv8.attn(c, over[:-64].view(5, 8, 128), one, start, out=over[64:].view(5, 8, 128))
    assert lib().rtxllm_kv8_append(c.ref, k.data_ptr(), 255, v.data_ptr(), 256, 0, None, one.data_ptr(), 1, 1, None) == 1
