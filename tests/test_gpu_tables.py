"""Page tables kept on the GPU (pages from a free list, positions and slots, pages given back) against a model that serves
the sequences one after the other. Whole numbers: everything is compared for equality, what must not change too."""
import numpy as np
import pytest

from test_gpu_pages import dev, host

pytestmark = pytest.mark.gpu

I32 = np.int32


def ceil(n, page):
    return -(-n // page)


class Model:
    def __init__(self, rng, lens, page, width, spare, total=None):
        self.page, self.width = page, width
        need = [max(0, ceil(n, page)) for n in lens]
        total = sum(need) + spare if total is None else total
        ids = rng.permutation(total).astype(I32)
        self.table = rng.integers(-5, total + 5, (len(lens), width)).astype(I32)  # whatever is behind a length
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.free = np.full(total, -7, I32)
        self.free[:total - at] = ids[at:]
        self.count, self.lens = total - at, np.array(lens, I32)

    def assign(self, add):
        cu, pos0, pos, slots = [0], [], [], []
        asked, begin = 0, self.count
        for b, n in enumerate(add):
            n, have = int(n), int(self.lens[b])
            ok = have >= 0 and n > 0 and have + n <= self.width * self.page
            held, need = ceil(have, self.page), 0
            if ok:
                need = ceil(have + n, self.page) - held
                asked += need
                ok = need == 0 or asked <= begin
            if ok:
                for i in range(need):
                    self.count -= 1
                    self.table[b, held + i] = self.free[self.count]
                for p in range(have, have + n):
                    pos.append(p)
                    slots.append(int(self.table[b, p // self.page]) * self.page + p % self.page)
                self.lens[b] += n
            pos0.append(have if ok else -1)
            cu.append(cu[-1] + (n if ok else 0))
        return np.array(cu, I32), np.array(pos0, I32), np.array(pos, I32), np.array(slots, I32)

    def release(self, keep):
        for b in reversed(range(len(keep))):
            if self.lens[b] < 0:
                continue
            n = min(max(int(keep[b]), 0), int(self.lens[b]))
            for i in reversed(range(ceil(n, self.page), ceil(int(self.lens[b]), self.page))):
                self.free[self.count] = self.table[b, i]
                self.count += 1
            self.lens[b] = n

    def on_device(self):
        return {"table": dev(self.table), "free": dev(self.free), "count": dev(np.array([self.count], I32)), "lens": dev(self.lens)}

    def check(self, d):
        assert int(host(d["count"])[0]) == self.count
        for n, want in (("table", self.table), ("lens", self.lens)):
            assert np.array_equal(host(d[n]), want), n
        assert np.array_equal(host(d["free"])[:self.count], self.free[:self.count])


def step(ctx, m, d, add, M=None):
    cu, pos0, pos, slots = m.assign(add)
    M = len(pos) if M is None else M
    p, s = dev(np.full(M, 99, I32)), dev(np.full(M, 99, I32))
    got = ctx.pages_assign(d["table"], m.page, d["free"], d["count"], d["lens"], dev(np.array(add, I32)), pos=p, slots=s)
    assert np.array_equal(host(got[0]), cu) and np.array_equal(host(got[1]), pos0)
    for x, want in ((p, pos), (s, slots)):
        full = np.full(M, -1, I32)
        full[:min(M, len(want))] = want[:M]
        assert np.array_equal(host(x), full)
    m.check(d)
    # the same places from the table alone
    if len(pos):
        p2, s2 = dev(np.full(len(pos) + 3, 99, I32)), dev(np.full(len(pos) + 3, 99, I32))
        ctx.pages_slots(d["table"], m.page, m.free.shape[0], got[0], got[1], pos=p2, slots=s2)
        assert np.array_equal(host(p2), np.append(pos, [-1] * 3)) and np.array_equal(host(s2), np.append(slots, [-1] * 3))
    return got


@pytest.mark.parametrize("B,page,most", [(1, 16, 1), (1, 8, 5000), (16, 64, 1), (37, 16, 200), (256, 16, 90), (257, 16, 90),
                                         (700, 16, 9), (1000, 8, 40), (1024, 16, 15), (1025, 32, 70), (3001, 16, 33), (16, 16, 1900),
                                         (40, 8, 1100)])
def test_assign_and_release(ctx, nnhip, B, page, most):
    print(f"tables B={B} page={page} most={most}", flush=True)
    rng = np.random.default_rng(B + page)
    lens = rng.integers(0, 300, B)
    lens[rng.random(B) < 0.2] = 0
    lens[rng.random(B) < 0.1] = -1
    width = ceil(300 + 3 * most, page)
    m = Model(rng, lens, page, width, B * ceil(most, page) * 2 + 5)
    d = m.on_device()
    for turn in range(4):
        add = rng.integers(0, most + 1, B)
        add[rng.random(B) < 0.1] = -3
        add[0] = most
        step(ctx, m, d, add, M=None if turn else int(np.maximum(add, 0).sum()) + 7)
        if turn % 2:
            keep = np.where(rng.random(B) < 0.3, 0, m.lens - rng.integers(-2, most + 1, B)).astype(I32)
            m.release(keep)
            ctx.pages_release(d["table"], page, d["free"], d["count"], d["lens"], dev(keep))
            m.check(d)


def test_release_takes_back(ctx, nnhip):
    """A release of what was given leaves the list, the count and the lengths as they were."""
    rng = np.random.default_rng(1)
    for B in (5, 300):
        m = Model(rng, rng.integers(0, 100, B), 16, 40, 10 * B)
        d = m.on_device()
        lens, free, count = m.lens.copy(), m.free.copy(), m.count
        step(ctx, m, d, rng.integers(0, 120, B))
        ctx.pages_release(d["table"], 16, d["free"], d["count"], d["lens"], dev(lens))
        assert np.array_equal(host(d["lens"]), lens) and int(host(d["count"])[0]) == count
        assert np.array_equal(host(d["free"])[:count], free[:count])


@pytest.mark.parametrize("B", [9, 400])
def test_scarce(ctx, nnhip, B):
    """More asked for than there is: sequences up to the last that fits, and later ones that need no page; then nothing."""
    rng = np.random.default_rng(2)
    m = Model(rng, rng.integers(0, 60, B), 16, 30, B)
    d = m.on_device()
    for _ in range(4):
        step(ctx, m, d, rng.integers(0, 60, B))
    m.count = 0
    d["count"].zero_()
    step(ctx, m, d, rng.integers(0, 5, B))


def test_table_limits(ctx, nnhip):
    """Sequences at their table's end, lengths and additions near 2^31, a count outside the list, no room for the tokens."""
    rng = np.random.default_rng(3)
    m = Model(rng, [60, 64, 0, 33, -2 ** 31, 5], 16, 4, 20)
    d = m.on_device()
    step(ctx, m, d, [4, 1, 2 ** 31 - 1, 32, 9, 59], M=10)
    d["lens"].copy_(dev(np.array([2 ** 31 - 1, 64, 0, 33, 3, 5], I32)))
    m.lens = host(d["lens"]).copy()
    step(ctx, m, d, [2 ** 31 - 1, -2 ** 31, 0, 0, 0, 0])
    for count, seen in ((-5, 0), (10 ** 6, m.free.shape[0])):
        m2 = Model(rng, [0, 0], 16, 4, 8)
        d = m2.on_device()
        d["count"].fill_(count)
        m2.count = min(seen, 8)
        step(ctx, m2, d, [20, 20])


def test_slots(ctx, nnhip):
    """Packed tokens of no sequence, positions past the table or below 0, pages outside the pool."""
    table = dev(np.array([[3, -1, 9, 5], [1, 2, 40, 0]], I32))
    cu, pos0 = dev(np.array([2, 30, 60], I32)), dev(np.array([20, 30], I32))
    pos, slots = dev(np.zeros(70, I32)), dev(np.zeros(70, I32))
    ctx.pages_slots(table, 16, 10, cu, pos0, pos=pos, slots=slots)
    want_p = np.full(70, -1)
    want_p[2:30], want_p[30:60] = np.arange(20, 48), np.arange(30, 60)
    assert np.array_equal(host(pos), want_p)
    ids = host(table)
    want = np.full(70, -1)
    for m in range(2, 60):
        i = ids[0 if m < 30 else 1, want_p[m] // 16]
        if 0 <= i < 10:
            want[m] = i * 16 + want_p[m] % 16
    assert np.array_equal(host(slots), want)
    only = dev(np.zeros(70, I32))
    ctx.pages_slots(table, 16, 10, cu, dev(np.array([-4, 50], I32)), pos=only)
    got = host(only)
    assert np.all(got[2:30] == -1) and np.array_equal(got[30:44], np.arange(50, 64)) and np.all(got[44:] == -1)


def test_captured_steps(ctx, nnhip):
    """Steps of a server in a graph: each replay goes on where the last one ended, as eager steps do."""
    import torch
    for B in (6, 300):
        rng = np.random.default_rng(4)
        m = Model(rng, rng.integers(0, 100, B), 16, 60, 4 * B)
        d, add = m.on_device(), dev(np.ones(B, I32))
        cu, pos0 = dev(np.zeros(B + 1, I32)), dev(np.zeros(B, I32))
        pos, slots = dev(np.zeros(B, I32)), dev(np.zeros(B, I32))
        side = torch.cuda.Stream()

        def call():
            ctx.pages_assign(d["table"], 16, d["free"], d["count"], d["lens"], add, cu=cu, pos0=pos0, pos=pos, slots=slots)

        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        m.assign(np.ones(B, int))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call()
        torch.cuda.synchronize()
        for _ in range(5):
            g.replay()
            torch.cuda.synchronize()
            want = m.assign(np.ones(B, int))
            m.check(d)
            assert np.array_equal(host(cu), want[0]) and np.array_equal(host(pos0), want[1])
            full = np.full(B, -1, I32)
            full[:len(want[3])] = want[3]
            assert np.array_equal(host(slots), full)


def test_table_refusals(ctx, nnhip):
    t, free, one, b = dev(np.zeros((2, 4), I32)), dev(np.zeros(8, I32)), dev(np.zeros(1, I32)), dev(np.zeros(2, I32))
    for page in (4, 12, 2048):
        with pytest.raises(nnhip.NNHipError, match="page_size"):
            ctx.pages_assign(t, page, free, one, b, b)
        with pytest.raises(nnhip.NNHipError, match="page_size"):
            ctx.pages_release(t, page, free, one, b, b)
    with pytest.raises(nnhip.NNHipError, match="shape"):
        ctx.pages_assign(t, 16, free, one, one, b)
    with pytest.raises(nnhip.NNHipError, match="shape"):
        ctx.pages_assign(t, 16, free, b, b, b)
    with pytest.raises(nnhip.NNHipError, match="dtype"):
        ctx.pages_release(t, 16, free, one, b, b.float())
    with pytest.raises(nnhip.NNHipError, match="null pointer"):
        nnhip._check(nnhip.lib().nnhip_pages_slots(ctx.h, t.data_ptr(), 4, 16, 8, None, None, 2, 5, None, None), "slots")
    with pytest.raises(nnhip.NNHipError, match="rows"):
        ctx.pages_slots(t, 16, 8, dev(np.zeros(4, I32)), pos=b)
    for call in (lambda x: ctx.pages_assign(x, 16, free, one, b, b), lambda x: ctx.pages_release(x, 16, free, one, b, b),
                 lambda x: ctx.pages_slots(x, 16, 8, dev(np.zeros(3, I32)), pos=b)):
        with pytest.raises(nnhip.NNHipError, match="page table must be"):
            call(dev(np.zeros(8, I32)))
