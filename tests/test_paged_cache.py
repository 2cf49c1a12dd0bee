"""The paged cache (scalablevectorsearch_amd.PagedCache, svsx_cache_*): page operations against a model of them in plain Python, refusals, capture."""
import ctypes as C
import random

import pytest

from scalablevectorsearch_amd import _lib


# ---- refusals: no GPU needed -------------------------------------------------------------------------------------------------------------------


def _desc(**changes):
    one = C.c_void_p(256)  # never followed: a refusal comes before any device work
    d = _lib.CacheDesc(C.sizeof(_lib.CacheDesc), 0, 1, 2, 10, 2, 4, 8, 8, 3, 5, one, one, one, one, one, one)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("changes, message", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=2), "row dtype"), (dict(dtype=9), "row dtype"), (dict(n_pages=0), "empty"), (dict(page_size=0), "empty"),
    (dict(key_dim=0), "empty"), (dict(n_pages=1 << 31), "2^31"), (dict(n_sequences=0), "n_sequences"), (dict(n_sequences=4097), "n_sequences"),
    (dict(max_pages=1 << 30), "max_pages"), (dict(max_pages=0), "max_pages"), (dict(page_size=1 << 20, max_pages=1 << 20), "max_pages"),
    (dict(n_sequences=4096, max_pages=1 << 20), "n_sequences"), (dict(d_keys=None), "null"), (dict(d_failures=None), "null"), (dict(d_values=None), "value_dim"),
    (dict(value_dim=0), "value_dim"),
])
def test_a_description_that_is_no_cache_is_refused(changes, message):
    _lib.build()
    L = _lib.lib()
    size = C.c_size_t()
    assert L.svsx_cache_workspace(C.byref(_desc(**changes)), 1, C.byref(size)) == _lib.INVALID_ARGUMENT
    assert message in L.svsx_last_error().decode()


def test_calls_check_their_arguments_before_any_device_work():
    _lib.build()
    L = _lib.lib()
    d, size = C.byref(_desc()), C.c_size_t()
    assert L.svsx_cache_workspace(d, 3, C.byref(size)) == _lib.SUCCESS and size.value > 0
    assert L.svsx_cache_workspace(None, 3, C.byref(size)) == _lib.NOT_INITIALIZED
    assert L.svsx_cache_workspace(d, 4097, C.byref(size)) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_extend_device(d, None, 256, 1, 1, 256, 256, size.value, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_extend_device(d, 256, 256, 3, 1, None, 256, size.value, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_extend_device(d, 256, 256, 3, 1, 256, 256, size.value - 1, None) == _lib.INVALID_ARGUMENT
    assert b"workspace" in L.svsx_last_error()
    assert L.svsx_cache_extend_device(d, 256, 256, 3, 1, 256, None, size.value, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_extend_device(d, None, None, 0, 0, None, None, 0, None) == _lib.SUCCESS       # nothing to do
    assert L.svsx_cache_copy_device(d, 256, None, 3, 0, 256, size.value, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_copy_device(d, None, None, 0, 0, None, 0, None) == _lib.SUCCESS
    assert L.svsx_cache_free_device(d, None, 1, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_free_device(d, None, 0, None) == _lib.SUCCESS
    assert L.svsx_cache_compact_device(d, None, 256, size.value, None) == _lib.INVALID_ARGUMENT
    assert L.svsx_cache_write_device(d, 2, 256, 1, 256, 16, 8, 256, 16, 8, None) == _lib.INVALID_ARGUMENT  # no such layer
    assert L.svsx_cache_write_device(d, 0, 256, 1, 256, 16, 8, None, 16, 8, None) == _lib.INVALID_ARGUMENT  # values missing
    assert L.svsx_cache_write_device(d, 0, None, 0, None, 0, 0, None, 0, 0, None) == _lib.SUCCESS


def test_threads_call_one_after_another(monkeypatch):
    """two calls of one cache are never in the library at once, where the launches of one could come between those of the other; two caches' may be"""
    import threading
    import time

    import torch

    from scalablevectorsearch_amd import cache as module

    class Library:
        """stands in for libsvsx.so and notes, per cache, calls that overlap"""

        inside, calls, overlaps = {}, 0, 0

        def svsx_cache_workspace(self, at, n, size):
            size._obj.value = 64
            return _lib.SUCCESS

        def call(self, at, *args):
            self.inside[at] = self.inside.get(at, 0) + 1
            self.overlaps += self.inside[at] > 1
            self.calls += 1
            time.sleep(0.002)
            self.inside[at] -= 1
            return _lib.SUCCESS

        svsx_cache_extend_device = svsx_cache_write_device = svsx_cache_copy_device = svsx_cache_free_device = svsx_cache_compact_device = call

    library = Library()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(module, "_on_device", lambda *a: None)
    monkeypatch.setattr(module, "_stream", lambda index: 0)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    caches = [module.PagedCache.from_device(torch.zeros(1, 4, 1, 2, 3), None, zeros(2, 2), zeros(2), zeros(4)) for _ in range(2)]
    monkeypatch.setattr(module, "paged_attention", lambda q, keys, *a, **k: library.call(next(c._at for c in caches if c.keys.data_ptr() == keys.data_ptr())))
    one, two, slots = zeros(1), zeros(2), torch.zeros(1, dtype=torch.int64)

    def work(c):
        for _ in range(3):
            c.extend(one, two, 1)
            c.write(slots, torch.zeros(1, 1, 3))
            c.fork(one, one)
            c.copy(one, one)
            c.free(one)
            c.compact()
            c.attend(torch.zeros(1, 1, 3))

    threads = [threading.Thread(target=work, args=(caches[i % 2],)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert library.calls == 6 * 21 and library.overlaps == 0


# ---- the model ---------------------------------------------------------------------------------------------------------------------------------


class Model:
    """What include/svsx.h says, in Python lists: rows are numbers that name the row that was written."""

    def __init__(self, layers, pages, page, sequences, columns):
        self.page, self.columns = page, columns
        self.rows = [[[None] * page for _ in range(pages)] for _ in range(layers)]
        self.table = [[-1] * columns for _ in range(sequences)]
        self.lengths, self.refs, self.failures = [0] * sequences, [0] * pages, 0

    def _firsts(self, seqs):
        return [0 <= s < len(self.lengths) and seqs.index(s) == i for i, s in enumerate(seqs)]

    def _take(self, need):
        """pages of each entry, None where refused: an entry is served while the sum of all needs up to it fits"""
        free, run, got = [p for p, r in enumerate(self.refs) if r == 0], 0, []
        for n in need:
            run += n
            got.append(None if n and run > len(free) else free[run - n:run])
        return got

    def extend(self, seqs, offsets, n_tokens):
        slots = [-1] * n_tokens
        ok = offsets[0] >= 0 and offsets[-1] <= n_tokens and all(a <= b for a, b in zip(offsets, offsets[1:]))
        fit, need = [], []
        for i, (s, first) in enumerate(zip(seqs, self._firsts(seqs))):
            have = new = 0
            if ok and first:
                have, new = -(-self.lengths[s] // self.page), -(-(self.lengths[s] + offsets[i + 1] - offsets[i]) // self.page)
            fit.append(ok and first and new <= self.columns)
            need.append(new - have if fit[-1] else 0)
        for i, (s, f, pages) in enumerate(zip(seqs, fit, self._take(need))):
            if not f or pages is None:
                self.failures += 1
                continue
            have = -(-self.lengths[s] // self.page)
            self.table[s][have:have + len(pages)] = pages
            for p in pages:
                self.refs[p] = 1
            for t in range(offsets[i], offsets[i + 1]):
                at = self.lengths[s] + t - offsets[i]
                slots[t] = self.table[s][at // self.page] * self.page + at % self.page
            self.lengths[s] += offsets[i + 1] - offsets[i]
        return slots

    def write(self, slots, names, layer):
        for s, name in zip(slots, names):
            if 0 <= s < len(self.refs) * self.page:
                self.rows[layer][s // self.page][s % self.page] = name

    def copy(self, sources, targets, share):
        n, fit, need = len(self.lengths), [], []
        for s, t, first in zip(sources, targets, self._firsts(targets)):
            good = first and 0 <= s < n and s not in targets and self.lengths[t] == 0
            fit.append(good)
            need.append(0 if not good else int(self.lengths[s] % self.page != 0) if share else -(-self.lengths[s] // self.page))
        taken = self._take(need)
        for s, t, f, pages in zip(sources, targets, fit, taken):
            if not f or pages is None:
                self.failures += 1
                continue
            whole = self.lengths[s] // self.page if share else 0
            for c in range(whole):
                self.table[t][c] = self.table[s][c]
                self.refs[self.table[s][c]] += 1
            for k, p in enumerate(pages):
                self.table[t][whole + k] = p
                self.refs[p] = 1
                for r in range(min(self.page, self.lengths[s] - (whole + k) * self.page)):
                    for layer in self.rows:
                        layer[p][r] = layer[self.table[s][whole + k]][r]
            self.lengths[t] = self.lengths[s]

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.lengths):
                self.failures += 1
                continue
            for c in range(-(-self.lengths[s] // self.page)):
                self.refs[self.table[s][c]] -= 1
                self.table[s][c] = -1
            self.lengths[s] = 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        moved = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        for to, p in zip(holes, [p for p in range(used, len(self.refs)) if self.refs[p] > 0]):
            moved[p] = to
            self.refs[to], self.refs[p] = self.refs[p], 0
            for layer in self.rows:
                layer[to] = list(layer[p])
        self.table = [[moved[p] if p >= 0 else -1 for p in row] for row in self.table]
        return moved


def test_the_model_keeps_its_invariants():
    """shared pages are full, counts are the table's, free entries are -1: over a random run, on the CPU"""
    rng = random.Random(3)
    m = Model(1, 40, 4, 8, 9)
    for _ in range(400):
        _step(m, rng)
        held = [0] * 40
        for s, row in enumerate(m.table):
            pages = -(-m.lengths[s] // 4)
            assert all(p >= 0 for p in row[:pages]) and all(p == -1 for p in row[pages:])
            for c, p in enumerate(row[:pages]):
                held[p] += 1
                assert m.refs[p] == 1 or (c + 1) * 4 <= m.lengths[s]
        assert held == m.refs
    assert m.failures > 0


def _step(m, rng):
    """one random operation, its arguments now and then wrong: (name, arguments, result)"""
    n = len(m.lengths)
    some = lambda: [rng.randrange(-1, n + 1) for _ in range(rng.randrange(0, 5))]  # noqa: E731
    op = rng.choice(["extend", "extend", "extend", "copy", "fork", "free", "compact"])
    if op == "extend":
        seqs = some()
        cuts = [0]
        for _ in seqs:
            cuts.append(cuts[-1] + rng.choice([0, 1, 1, 2, m.page, 3 * m.page + 1]))
        total = cuts[-1] + rng.choice([0, 0, 2])
        if rng.random() < 0.05 and len(cuts) > 1:
            cuts[0] = cuts[-1] + 1
        args = (seqs, cuts, total)
        return op, args, m.extend(*args)
    if op in ("copy", "fork"):
        sources = some()
        targets = [rng.randrange(-1, n + 1) for _ in sources]
        return op, (sources, targets), m.copy(sources, targets, op == "fork")
    if op == "free":
        args = (some(),)
        return op, args, m.free(*args)
    return op, (), m.compact()


# ---- the kernels against the model -----------------------------------------------------------------------------------------------------------------


def _same(cache, m, heads, key_dim, value_dim):
    import torch

    assert cache.table.tolist() == m.table and cache.lengths.tolist() == m.lengths and cache.refs.tolist() == m.refs and cache.failures.item() == m.failures
    names = torch.tensor([[[-1 if r is None else r for r in page] for page in layer] for layer in m.rows])  # layers, pages, rows
    known = names >= 0
    for x, dim in ((cache.keys, key_dim), (cache.values, value_dim)):
        if x is not None:
            want = _row(names, heads, dim).permute(0, 1, 3, 2, 4).to(x.dtype)  # layers, pages, heads, rows, dim
            assert torch.equal(x.cpu().masked_fill(~known[:, :, None, :, None], 0), want.masked_fill(~known[:, :, None, :, None], 0))


def _row(names, heads, dim):
    """the row that a name stands for: exact in 16 bits, other in every column and head"""
    import torch

    return (names[..., None, None] * 7 + torch.arange(heads)[:, None] * 31 + torch.arange(dim)) % 251


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, layers, pages, page, heads, key_dim, value_dim", [
    ("float16", 2, 40, 4, 2, 8, 8), ("bfloat16", 1, 40, 1, 3, 5, 7), ("float32", 3, 40, 3, 1, 6, 0), ("float16", 1, 33, 16, 2, 64, 32), ("bfloat16", 1, 20000, 2, 1, 2, 2),
])
def test_random_operations_leave_what_the_model_leaves(dtype, layers, pages, page, heads, key_dim, value_dim):
    import torch

    import scalablevectorsearch_amd as svs

    rng = random.Random(pages * page + heads)
    cache = svs.PagedCache(pages, page, heads, key_dim, value_dim, layers, getattr(torch, dtype), n_sequences=8, max_pages=9)
    m, name = Model(layers, pages, page, 8, 9), 0
    for step in range(60 if pages > 1000 else 150):
        op, args, want = _step(m, rng)
        lists = [torch.tensor(a, dtype=torch.int32, device="cuda") if isinstance(a, list) else a for a in args]
        got = getattr(cache, op)(*lists)
        if want is not None:
            assert got.tolist() == want, (step, op, args)
        if op == "extend" and args[2]:
            for layer in range(layers):
                names = torch.arange(name, name + args[2])
                name += args[2]
                rows = [_row(names, heads, d).to(cache.keys.dtype).cuda() if d else None for d in (key_dim, value_dim)]
                if layer == 1:  # rows of a wider array, heads outside tokens
                    rows = [x if x is None else torch.stack([x, x]).transpose(1, 2).contiguous()[1].transpose(0, 1) for x in rows]
                cache.write(got, rows[0], rows[1], layer=layer)
                m.write(want, names.tolist(), layer)
        if step % 10 == 9 or pages < 100:
            _same(cache, m, heads, key_dim, value_dim)
    _same(cache, m, heads, key_dim, value_dim)


@pytest.mark.gpu
def test_many_sequences_and_a_pool_that_is_exhausted():
    """4096 entries a call, prompts over many pages, more asked than there is: the first that does not fit and all that need pages behind it are refused"""
    import torch

    import scalablevectorsearch_amd as svs

    rng = random.Random(1)
    cache = svs.PagedCache(30000, 2, 1, 2, 0, dtype=torch.float32, n_sequences=4096, max_pages=64)
    m = Model(1, 30000, 2, 4096, 64)
    for _ in range(3):
        seqs = list(range(4096))
        rng.shuffle(seqs)
        cuts = [0]
        for _ in seqs:
            cuts.append(cuts[-1] + rng.choice([0, 1, 7, 17, 21]))
        want = m.extend(seqs, cuts, cuts[-1])
        got = cache.extend(torch.tensor(seqs, dtype=torch.int32).cuda(), torch.tensor(cuts, dtype=torch.int32).cuda(), cuts[-1])
        assert torch.equal(got.cpu(), torch.tensor(want))
        half = seqs[::2]
        m.free(half)
        cache.free(half)  # a list on the host
        _same(cache, m, 1, 2, 0)
    assert m.failures > 0


@pytest.mark.gpu
def test_a_step_is_captured_and_replayed():
    """free + fork + extend + write as one graph, replayed with other rows and the program's own work between the replays, equals the eager calls"""
    import torch

    import scalablevectorsearch_amd as svs

    def fresh():
        g = torch.Generator().manual_seed(5)
        cache = svs.PagedCache(64, 4, 2, 16, dtype=torch.float16, n_sequences=6, max_pages=10)
        slots = cache.extend([0, 1], torch.tensor([0, 13, 33], dtype=torch.int32).cuda(), 33)
        rows = torch.randn(33, 2, 16, generator=g).half().cuda()
        cache.write(slots, rows, -rows)
        return cache

    new = torch.zeros(4, 2, 16, dtype=torch.float16, device="cuda")
    src, dst, off = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 0, 1, 1], [2, 3, 4, 5], [0, 1, 2, 3, 4]))

    def step(cache):
        cache.free(dst)
        cache.fork(src, dst)
        cache.write(cache.extend(dst, off, 4), new, new + 1)
        return cache.compact()

    cache, eager = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    step(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moved = step(cache)
    for k in range(4):
        new.fill_(k + 1)
        graph.replay()
        want = step(eager)
        torch.randn(1000, device="cuda").sum().item()
        assert torch.equal(moved, want)
        for name in ("keys", "values", "table", "lengths", "refs", "failures"):
            assert torch.equal(getattr(cache, name), getattr(eager, name)), (k, name)


@pytest.mark.gpu
def test_threads_on_one_stream():
    """four threads fork, grow, write and free sequences of their own, a fifth compacts: in the end every sequence has its parent's rows and its own, and counts are the table's"""
    import threading

    import torch

    import scalablevectorsearch_amd as svs

    cache = svs.PagedCache(200, 4, 1, 2, 0, dtype=torch.float32, n_sequences=5, max_pages=9)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    parent = torch.arange(46, dtype=torch.float32, device="cuda").reshape(23, 1, 2)
    cache.write(cache.extend(ints(0), ints(0, 23), 23), parent)
    lists = [(ints(0), ints(k), ints(0, 2), torch.full((2, 1, 2), 100.0 + k, device="cuda")) for k in range(1, 5)]
    torch.cuda.synchronize()
    errors = []

    def work(zero, mine, two, rows):
        try:
            for _ in range(50):
                cache.free(mine)
                cache.fork(zero, mine)
                cache.extend(mine, two, 2)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    def compact():
        for _ in range(50):
            cache.compact()

    threads = [threading.Thread(target=work, args=x) for x in lists] + [threading.Thread(target=compact)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for _, mine, two, rows in lists:  # slots hold until the next compact: written here, to two more rows
        cache.write(cache.extend(mine, two, 2), rows)
    assert not errors and cache.failures.item() == 0 and cache.lengths.tolist() == [23, 27, 27, 27, 27]
    table, held = cache.table.cpu().long(), torch.zeros(200, dtype=torch.int32)
    for s in range(5):
        of = table[s, :-(-int(cache.lengths[s]) // 4)]
        held[of] += 1
        rows = cache.keys[0].cpu()[of, 0].reshape(-1, 2)
        assert torch.equal(rows[:23], parent[:, 0].cpu()) and (s == 0 or (rows[25:27] == 100 + s).all())
    assert torch.equal(held, cache.refs.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("length", [-1, -3, -4, -(2**31), 37, 2**31 - 1])
def test_a_length_that_no_sequence_has_is_refused(length):
    """lengths below zero and beyond the table (9 pages of 4 rows) in an adopted cache: the sequence neither grows nor is copied, nothing else changes, and the entries beside it are
    served"""
    import torch

    import scalablevectorsearch_amd as svs

    cache = svs.PagedCache(30, 4, 1, 2, 0, dtype=torch.float32, n_sequences=6, max_pages=9)
    cache.extend([0, 1], torch.tensor([0, 6, 15], dtype=torch.int32).cuda(), 15)
    cache.lengths[0] = length
    table, refs = cache.table.tolist(), cache.refs.tolist()
    for share in (False, True):
        (cache.fork if share else cache.copy)([0, 1], [2, 3])
        assert cache.failures.item() == 1 and cache.lengths.tolist() == [length, 9, 0, 9, 0, 0]
        assert cache.table[0].tolist() == table[0] and cache.table[2].tolist() == table[2] and cache.table[4:].tolist() == table[4:]
        assert sum(cache.refs.tolist()) == sum(refs) + 3
        cache.free([3])
        assert cache.refs.tolist() == refs and cache.table.tolist() == table
        cache.failures.zero_()
    slots = cache.extend([0, 4], torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), 2).tolist()
    assert cache.failures.item() == 1 and cache.lengths.tolist() == [length, 9, 0, 0, 1, 0] and slots[0] == -1 and slots[1] >= 0


@pytest.mark.gpu
def test_pages_beyond_two_to_the_31_elements():
    import torch

    import scalablevectorsearch_amd as svs

    pages = (1 << 31) // (16 * 128) + 5
    cache = svs.PagedCache(pages, 16, 1, 128, 0, dtype=torch.float16, n_sequences=2, max_pages=4)
    cache.refs[: pages - 3] = 1
    rows = torch.randn(17, 1, 128, device="cuda").half()
    slots = cache.extend([0], torch.tensor([0, 17], dtype=torch.int32).cuda(), 17)
    assert slots[0].item() == (pages - 3) * 16
    cache.write(slots, rows)
    assert torch.equal(cache.keys[0, pages - 3, 0], rows[:16, 0]) and torch.equal(cache.keys[0, pages - 2, 0, 0], rows[16, 0])
    cache.fork([0], [1])
    assert cache.table[1, :2].tolist() == [pages - 3, pages - 1] and torch.equal(cache.keys[0, pages - 1, 0, 0], rows[16, 0])
    assert cache.refs[-3:].tolist() == [2, 1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [(1 << 13) - 1, (1 << 16) + 3])
def test_writing_more_words_than_a_grid_has_threads(tokens):
    """65537 half-words a row: 2^29 of them, and more than 2^32; most slots are outside the cache, the rows that count are the first, the last and some between"""
    import torch

    import scalablevectorsearch_amd as svs

    cache = svs.PagedCache(4, 2, 1, 65537, 0, dtype=torch.float16, n_sequences=2, max_pages=2)
    row = torch.randn(1, 1, 65537, device="cuda").half()
    rows = row.expand(tokens, 1, 65537)  # every token's row is the same memory
    slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    for slot, token in ((0, 0), (5, tokens // 2), (6, tokens - 4), (7, tokens - 1)):
        slots[token] = slot
    slots[3] = 8  # outside, too
    cache.write(slots, rows)
    got = cache.keys[0, :, 0].reshape(8, 65537)
    for slot in range(8):
        assert torch.equal(got[slot], row[0, 0] if slot in (0, 5, 6, 7) else torch.zeros_like(row[0, 0])), slot


@pytest.mark.gpu
def test_wrong_arguments_are_refused():
    import torch

    import scalablevectorsearch_amd as svs

    cache = svs.PagedCache(8, 4, 2, 16, dtype=torch.float16, n_sequences=3)
    off, slots, rows = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), torch.zeros(1, 2, 16).half().cuda()
    bad = [
        lambda: svs.PagedCache(0, 4, 2, 16), lambda: svs.PagedCache(8, 4, 2, 16, dtype=torch.float64), lambda: svs.PagedCache(8, 4, 2, 16, n_sequences=5000),
        lambda: cache.extend([0, 1], off, 1), lambda: cache.extend(torch.zeros(1, dtype=torch.int64).cuda(), off, 1), lambda: cache.extend([0], off.cpu(), 1),
        lambda: cache.extend([0], off, -1), lambda: cache.copy([0], [1, 2]), lambda: cache.free(torch.zeros(1, 1, dtype=torch.int32).cuda()),
        lambda: cache.write(slots, rows), lambda: cache.write(slots, rows.float(), rows), lambda: cache.write(slots.int(), rows, rows),
        lambda: cache.write(slots, rows, rows[..., :8]), lambda: cache.write(slots, rows, rows, layer=1), lambda: cache.write(slots, rows.cpu(), rows),
        lambda: cache.write(slots, rows, rows.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: svs.PagedCache.from_device(cache.keys, cache.values, cache.table.long(), cache.lengths, cache.refs),
        lambda: svs.PagedCache.from_device(cache.keys, cache.values, cache.table, cache.lengths, cache.refs[1:]),
        lambda: svs.PagedCache.from_device(cache.keys[..., ::2], cache.values, cache.table, cache.lengths, cache.refs), lambda: cache.attend(rows, layer=1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(svs.SvsxError) as e:
            call()
        assert e.value.code == _lib.INVALID_ARGUMENT, i
    assert cache.lengths.sum().item() == 0 and cache.failures.item() == 0
