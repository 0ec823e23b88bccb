"""The operators of a serving step together, as a server of growing and shrinking sequences uses them: room in the paged caches
(paged_append), the write into them (rotary_axes_cached), the attention of the new tokens (paged_attention_chunk), the residual
row and the next norm (rms_norm_add), and the tokens that are taken back (paged_truncate).

The attention is held against its definition in 64 bits, over keys and values that the test keeps itself, with the tolerance of
test_gpu_chunk_attention; the norm against the separate calls, to the bit; lengths and free pages against a count of them."""
import pytest

from test_gpu_chunk_attention import _close, _cu, _ref
from test_gpu_mixers import _gen, _torch

pytestmark = pytest.mark.gpu

PAGE, EPS, LEFT = 16, 1e-6, 7.0


class _Server:
    def __init__(self, mcv, cuda, B, width, pages, Hq, Hkv, D, rows, seed):
        torch = _torch()
        self.mcv, self.cuda, self.gen = mcv, cuda, _gen(seed)
        self.B, self.Hq, self.Hkv, self.D, self.pages = B, Hq, Hkv, D, pages
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=cuda)
        self.lens = torch.zeros(B, dtype=torch.int32, device=cuda)
        self.free = torch.randperm(pages, generator=self.gen).int().to(cuda)
        self.count = torch.tensor([pages], dtype=torch.int32, device=cuda)
        self.kc, self.vc = (torch.full((pages, PAGE, Hkv, D), float("nan"), device=cuda).half() for _ in range(2))
        self.freq, self.axis = mcv.rotary_axes_table(64, 1e6, (12, 10, 10), device=cuda)
        self.gamma = torch.randn(Hq * D, generator=self.gen).half().to(cuda)
        half = lambda *s: torch.zeros(*s, dtype=torch.float16, device=cuda)      # noqa: E731
        self.q, self.k, self.v = half(rows, Hq, D), half(rows, Hkv, D), half(rows, Hkv, D)
        self.x = half(rows, Hq * D)
        self.cu = torch.zeros(B + 1, dtype=torch.int32, device=cuda)
        self.slots, self.places = (torch.zeros(rows, dtype=torch.int64, device=cuda) for _ in range(2))
        self.rotated, self.out, self.normed, self.summed = half(rows, Hq, D), half(rows, Hq, D), half(rows, Hq * D), half(rows, Hq * D)
        self.held = [[torch.zeros(0, Hkv, D).half() for _ in range(2)] for _ in range(B)]

    def inputs(self, n):
        torch = _torch()
        for t in (self.q, self.k, self.v, self.x):
            t.copy_(torch.randn(t.shape, generator=self.gen).half())
        self.cu.copy_(_cu(n))
        self.out.fill_(LEFT)

    def step(self):
        mcv = self.mcv
        mcv.paged_append(self.table, self.lens, self.cu, PAGE, free_pages=self.free, free_count=self.count, slots=self.slots, positions=self.places)
        mcv.rotary_axes_cached(self.q, self.k, self.v, self.places.expand(3, -1).contiguous(), self.freq, self.axis, self.kc, self.vc, self.slots,
                               q_out=self.rotated)
        mcv.paged_attention_chunk(self.rotated, self.kc, self.vc, self.table, self.lens, self.cu, out=self.out)
        mcv.rms_norm_add(self.out.flatten(1), self.x, self.gamma, EPS, out=self.normed, residual_out=self.summed)

    def check(self, n):
        torch, mcv = _torch(), self.mcv
        torch.cuda.synchronize()
        places = torch.cat([torch.arange(m) + len(k) for m, (k, _) in zip(n, self.held)] + [torch.zeros(len(self.q) - sum(n), dtype=torch.int64)])
        assert (self.places.cpu() == places).all()
        turned = mcv.rotary_axes(self.q, self.k, places.expand(3, -1).contiguous().to(self.cuda), self.freq, self.axis)
        assert (turned[0] == self.rotated).all()
        k, v, first = turned[1].cpu(), self.v.cpu(), 0
        for b, m in enumerate(n):
            self.held[b] = [torch.cat((old, new[first:first + m])) for old, new in zip(self.held[b], (k, v))]
            first += m
        self.lengths()
        out = self.out.cpu()
        _close(out[:first], _ref(self.rotated.cpu()[:first], self.held, n, [len(x) for x, _ in self.held], self.D ** -0.5))
        assert (out[first:] == LEFT).all()
        total = (self.out.flatten(1).float() + self.x.float()).half()
        assert (self.summed == total).all() and (self.normed == mcv.rms_norm(total, self.gamma, EPS)).all()

    def keep(self, keep):
        torch = _torch()
        self.mcv.paged_truncate(self.table, self.lens, torch.tensor(keep, dtype=torch.int32, device=self.cuda), PAGE, self.free, self.count)
        self.held = [[t[:m] for t in kv] for kv, m in zip(self.held, keep)]
        self.lengths()

    def lengths(self):
        torch = _torch()
        torch.cuda.synchronize()
        lens = [len(k) for k, _ in self.held]
        assert self.lens.tolist() == lens
        used = [self.table[b, :-(-m // PAGE)].tolist() for b, m in enumerate(lens)]
        free = self.free[:int(self.count)].tolist()
        assert sorted(sum(used, free)) == list(range(self.pages))           # every page has one place


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (4, 4, 128), (8, 1, 256)])
def test_a_run(mcv, cuda, Hq, Hkv, D):
    """Prompts, single tokens, drafts of which some are taken back, a sequence that ends and another in its place."""
    s = _Server(mcv, cuda, 5, 24, 70, Hq, Hkv, D, 300, 1)
    for n, keep in (([70, 5, 0, 33, 1], None), ([1, 1, 1, 1, 1], None), ([4, 4, 4, 4, 4], [-3, 0, -2, -1, -4]), ([1, 200, 16, 15, 0], None),
                    ([1, 0, 1, 1, 1], [0, -999, 0, 0, 0]), ([2, 130, 1, 60, 90], None), ([1, 1, 1, 1, 1], [-999] * 5), ([300, 0, 0, 0, 0], None)):
        s.inputs(n)
        s.step()
        s.check(n)
        if keep is not None:
            s.keep([max(0, len(k) + m) for m, (k, _) in zip(keep, s.held)])


def test_in_a_graph(mcv, cuda):
    """One step captured and replayed over drafts, prompts and nothing at all, with eager work between."""
    torch = _torch()
    s = _Server(mcv, cuda, 4, 40, 120, 8, 2, 128, 200, 2)
    s.inputs([0, 0, 0, 0])
    s.step()                                     # (of no token: lengths stay)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.step()
    for i, n in enumerate(([100, 50, 0, 50], [1, 1, 1, 1], [4, 4, 190, 2], [0, 0, 0, 0], [1, 1, 1, 1], [5, 150, 5, 40])):
        s.inputs(n)
        graph.replay()
        s.check(n)
        if i % 2:
            s.keep([max(0, len(k) - i) for k, _ in s.held])


# ------------------------------------------------------------------------- the attention's workspace --
def _several(cuda, seed=3):
    """Calls whose tiles are in one, up to four, and more parts."""
    from test_gpu_chunk_attention import _case
    cases = ([60], [0], 8, 2, 128), ([300], [90], 8, 2, 256), ([700], [0], 8, 2, 256), ([3, 40], [6000, 900], 8, 2, 64), ([1] * 9, [4000] * 9, 8, 2, 128)
    return [[x.to(cuda) for x in _case(seed + i, n, held, Hq, Hkv, D, 32)[:6]] for i, (n, held, Hq, Hkv, D) in enumerate(cases)]


def test_its_counters_end_at_zero(mcv, cuda):
    torch = _torch()
    calls = _several(cuda)
    want = [mcv.paged_attention_chunk(*a) for a in calls]
    for _ in range(5):                           # and who is last changes no bit
        assert all((mcv.paged_attention_chunk(*a) == w).all() for a, w in zip(calls, want))
    torch.cuda.synchronize()
    held = list(mcv.mixers._CHUNK_WS.values())
    assert held and all((ws[:mcv.mixers._CHUNK_COUNTER_BYTES] == 0).all() for ws in held)


def test_given_a_workspace_of_its_own(mcv, cuda):
    """Through the C interface: none (nothing is cut), the bytes it asks for and not one more, and those of a larger call."""
    torch = _torch()
    lib, stream = mcv.lib(), torch.cuda.current_stream().cuda_stream
    for a in _several(cuda):
        q, k, v, table, lens, cu = a
        (T, Hq, D), (pages, page, Hkv, _), (B, width) = q.shape, k.shape, table.shape
        want = mcv.paged_attention_chunk(*a)
        least = lib.mcv_paged_attention_chunk_workspace_bytes(B, T, Hq, Hkv, D, width * page)
        most = lib.mcv_paged_attention_chunk_workspace_bytes(B, 9 * T, Hq, Hkv, D, 1 << 20)
        assert most >= least
        for nbytes in (0, least, most):
            ws = torch.zeros(max(nbytes, 256) + 4096, dtype=torch.uint8, device=cuda)
            ws[nbytes:] = 91
            for _ in range(2):
                out = torch.full_like(q, LEFT)
                rc = lib.mcv_paged_attention_chunk(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], pages,
                                                   page, table.data_ptr(), table.stride(0), width, lens.data_ptr(), width * page, cu.data_ptr(), B, T, Hq, Hkv,
                                                   D, D ** -0.5, out.data_ptr(), ws.data_ptr() if nbytes else None, nbytes, stream)
                assert rc == 0
                torch.cuda.synchronize()
                # cut or not, a sum of the same weights in 32 bits, rounded once: at most a step of fp16 apart
                assert ((out.float() - want.float()).abs() <= 2.0 ** -9 * want.float().abs() + 2.0 ** -9).all()
                if nbytes:
                    assert (out == want).all()
            assert (ws[nbytes:] == 91).all() and (ws[:min(nbytes, 8192)] == 0).all()


@pytest.mark.parametrize("B", [1, 3, 64, 65, 700])
def test_offsets_that_fall(mcv, cuda, B):
    """Rows would have two sequences: none is written, and the next call finds the workspace as it was."""
    torch = _torch()
    a = _several(cuda)[2]
    want = mcv.paged_attention_chunk(*a)
    T = len(a[0])
    cu = torch.linspace(0, T, B + 1, device=cuda).int()
    cu[B // 2:] = cu[B // 2:].flip(0)
    table, lens = a[3].expand(B, -1).contiguous(), a[4].expand(B).contiguous()
    out = torch.full_like(a[0], LEFT)
    mcv.paged_attention_chunk(*a[:3], table, lens, cu, out=out)
    assert (out == LEFT).all()
    assert (mcv.paged_attention_chunk(*a) == want).all()
    torch.cuda.synchronize()
    assert all((ws[:mcv.mixers._CHUNK_COUNTER_BYTES] == 0).all() for ws in mcv.mixers._CHUNK_WS.values())


def test_more_sequences_than_threads(mcv, cuda):
    """1500 sequences, some without new tokens, some with one and a few with many, in a batch with rows of no sequence."""
    from test_gpu_chunk_attention import _case
    torch = _torch()
    n = [(0, 1, 1, 2, 5)[i % 5] if i % 400 else 90 for i in range(1500)]
    held = [(7 * i) % 70 if i % 311 else 700 for i in range(1500)]
    q, k, v, table, lens, cu, kv = _case(8, n, held, 4, 2, 64, 16)
    q = torch.cat((q, q[:9]))
    out = torch.full_like(q, LEFT).to(cuda)
    mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)), out=out)
    _close(out[:sum(n)], _ref(q[:sum(n)], kv, n, lens.tolist(), 64 ** -0.5))
    assert (out[sum(n):] == LEFT).all()


def test_one_size_a_stream(mcv, cuda):
    torch = _torch()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in _several(cuda):
            mcv.paged_attention_chunk(*a)
        held = [ws.numel() for (_, stream, _), ws in mcv.mixers._CHUNK_WS.items() if stream == side.cuda_stream]
    side.synchronize()
    assert held == [mcv.mixers.CHUNK_WORKSPACE_BYTES]


def test_streams_at_once(mcv, cuda):
    torch = _torch()
    calls = _several(cuda)
    want = [mcv.paged_attention_chunk(*a) for a in calls]
    outs = [[torch.empty_like(w) for w in want] for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        for i in range(len(calls)):
            for j, stream in enumerate(streams):
                x = (i + j) % len(calls)
                mcv.paged_attention_chunk(*calls[x], out=outs[j][x], stream=stream)
    torch.cuda.synchronize()
    assert all((got == w).all() for out in outs for got, w in zip(out, want))


def test_graphs_at_once(mcv, cuda):
    """Two graphs, captured one after the other on one stream, replayed on two streams and after one another."""
    torch = _torch()
    calls = _several(cuda)
    want = [mcv.paged_attention_chunk(*a) for a in calls]
    side, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for order in (calls, calls[::-1]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append([mcv.paged_attention_chunk(*a) for a in order])
        graphs.append(graph)
    outs[1].reverse()
    for turn in range(6):
        for out in outs:
            for t in out:
                t.fill_(LEFT)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, others if turn % 2 else (side, side)):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = mcv.paged_attention_chunk(*calls[turn % len(calls)])
        torch.cuda.synchronize()
        assert (eager == want[turn % len(calls)]).all()
        assert all((got == w).all() for out in outs for got, w in zip(out, want)), turn


def test_calls_allocate_nothing(mcv, cuda):
    """Given their outputs, and once the stream has its workspace."""
    torch = _torch()
    calls = [(a, torch.empty_like(a[0])) for a in _several(cuda)]
    s = _Server(mcv, cuda, 3, 8, 24, 8, 2, 64, 40, 4)
    keep = torch.zeros(3, dtype=torch.int32, device=cuda)

    def once():
        for a, out in calls:
            mcv.paged_attention_chunk(*a, out=out)
        mcv.paged_append(s.table, s.lens, s.cu, PAGE, free_pages=s.free, free_count=s.count, slots=s.slots, positions=s.places)
        mcv.paged_truncate(s.table, s.lens, keep, PAGE, s.free, s.count)
        mcv.rms_norm_add(s.x, s.x, s.gamma, EPS, out=s.normed, residual_out=s.summed)

    s.cu.copy_(_cu([20, 5, 10]))
    once()
    torch.cuda.synchronize()
    asked = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]    # noqa: E731
    before = asked()
    for _ in range(3):
        once()
    assert asked() == before
    torch.cuda.synchronize()


def test_outputs_of_another_stream(mcv, cuda):
    """What a call on another stream allocates is that stream's: freed at once, the current stream does not get it."""
    torch = _torch()
    side = torch.cuda.Stream()
    a = _several(cuda)[3]
    s = _Server(mcv, cuda, 3, 8, 24, 8, 2, 64, 40, 5)
    s.inputs([20, 5, 15])
    lens = torch.zeros_like(s.lens)
    calls = [
        lambda **on: (mcv.paged_attention_chunk(*a, **on),),
        lambda **on: mcv.rms_norm_add(s.x, s.x, s.gamma, EPS, **on),
        lambda **on: mcv.rms_norm_add_w8a8_quantize(s.x, s.x, s.gamma, EPS, **on)[:3],
        lambda **on: mcv.paged_append(s.table.clone(), s.lens, s.cu, PAGE, tokens=40, free_pages=s.free, free_count=s.count.clone(), seq_lens_out=lens, **on)[:2],
    ]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        got = call(stream=side)
        side.synchronize()
        assert all((x == y).all() for x, y in zip(got, want))
        where, shapes = {t.data_ptr() for t in got}, [(t.shape, t.dtype) for t in got]
        del got
        fresh = [torch.empty(shape, dtype=dtype, device=cuda) for shape, dtype in shapes]
        assert not where & {t.data_ptr() for t in fresh}
