"""PagedSequences: the oracle's own rules, and the refusals that need no GPU."""
import contextlib
import copy
import importlib
import pickle
import random
import struct

import pytest
import torch

from oracle.pages_ref import PagedSequencesRef

pages = importlib.import_module("nanokv-llm_amd.engine.pages")
_lib = importlib.import_module("nanokv-llm_amd._lib")
P = 0x10000


def test_oracle_keeps_counts_tables_and_contents():
    """Random programs: counts are the tables' entries, a partly filled page has one holder, and
    every row reads back the tokens that were written for it, whatever was moved or copied."""
    rng = random.Random(1)
    B, S = 4, 7
    ref = PagedSequencesRef(torch.zeros(2, 1, 25, B, 1, 1, dtype=torch.int64), S, 6)
    want, clock = [[] for _ in range(S)], 0
    for _ in range(600):
        rows = rng.sample(range(S), rng.randint(1, 4))
        op = rng.choice(["append", "append", "truncate", "fork", "copy", "compact"])
        if op == "append":
            n = [rng.randint(0, 9) for _ in rows]
            cu = [sum(n[:i]) for i in range(len(n) + 1)]
            slots, ok = ref.append(rows, cu=cu, n_tokens=cu[-1])
            for i, r in enumerate(rows):
                for t in slots[cu[i]:cu[i + 1]]:
                    clock += 1
                    assert (t >= 0) == bool(ok[i])
                    if ok[i]:
                        ref.kv.view(2, -1)[:, t] = clock
                        want[r].append(clock)
        elif op == "truncate":
            keep = [rng.randint(0, ref.lens[r]) for r in rows]
            for r, k, ok in zip(rows, keep, ref.truncate(rows, keep)):
                want[r] = want[r][:k] if ok else want[r]
        elif op == "compact":
            ref.compact(rng.choice([1, 3, 25]))
        else:
            parents = [rng.randrange(S) for _ in rows]
            before = [list(want[p]) for p in parents]
            for r, b, ok in zip(rows, before, ref.fork(parents, rows, op == "fork")):
                want[r] = b if ok else want[r]
        held = [x for t in ref.tables for x in t if x >= 0]
        assert ref.refs == [held.count(x) for x in range(25)]
        for r in range(S):
            n = ref.lens[r]
            assert [x >= 0 for x in ref.tables[r]] == [j * B < n for j in range(6)]
            got = [int(ref.kv[0, 0, ref.tables[r][t // B], t % B]) for t in range(n)]
            assert got == want[r] and n == len(want[r])
            assert n % B == 0 or ref.refs[ref.tables[r][n // B]] == 1


def test_constructor_refuses_bad_pools_and_states():
    kv = torch.zeros(2, 1, 4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="expected GPU"):
        pages.PagedSequences(kv, 2, 2)
    with pytest.raises(ValueError, match="contiguous"):
        pages.PagedSequences(kv.transpose(2, 3), 2, 2)
    with pytest.raises(ValueError, match="contiguous"):
        pages.PagedSequences(kv[0], 2, 2)


def _args(**kw):
    a = dict(kv=P, planes=4, pages=10, block=16, row=256, refs=P, lens=P, tables=P, stride=8,
             width=8, rows=5, ws=P, wsb=1 << 30)
    a.update(kw)
    return struct.pack("13q", *a.values())


BAD = [
    (dict(planes=0), -1, b"bad sizes"), (dict(pages=0), -1, b"bad sizes"),
    (dict(block=0), -1, b"bad sizes"), (dict(rows=0), -1, b"bad sizes"),
    (dict(stride=7), -1, b"bad sizes"), (dict(row=24), -4, b"multiple of 16"),
    (dict(rows=8193), -4, b"at most"), (dict(pages=(1 << 20) + 1), -4, b"at most"),
    (dict(planes=65536), -4, b"at most"), (dict(pages=1 << 20, block=2048), -4, b"32 bits"),
    (dict(width=1 << 28, stride=1 << 28), -4, b"32 bits"), (dict(row=1 << 32), -4, b"32 bits"),
    (dict(kv=0), -1, b"null"), (dict(refs=0), -1, b"null"), (dict(lens=0), -1, b"null"),
    (dict(tables=0), -1, b"null"), (dict(kv=P + 8), -1, b"aligned"),
    (dict(refs=P + 4), -1, b"aligned"), (dict(ws=0), -3, b"workspace"),
    (dict(ws=P + 8), -3, b"workspace"), (dict(wsb=1000), -3, b"workspace"),
]


@pytest.mark.parametrize("kw,code,msg", BAD)
def test_entry_points_refuse_bad_pages(kw, code, msg):
    lib = _lib.lib()
    a = _args(**kw)
    for rc in (lib.nkv_pages_append(a, P, 1, None, 1, P, P, None),
               lib.nkv_pages_truncate(a, P, P, 1, None, 0, P, None),
               lib.nkv_pages_fork(a, P, P, 1, 1, P, None),
               lib.nkv_pages_compact(a, 1, P, P, None)):
        assert rc == code and msg in lib.nkv_last_error(), lib.nkv_last_error()


@pytest.mark.parametrize("call,args,code,msg", [
    ("append", (P, -1, None, -1, P, P), -1, b"rows"),
    ("append", (P, 8193, None, 8193, P, P), -1, b"rows"),
    ("append", (P, 3, None, 4, P, P), -1, b"one token a row"),
    ("append", (P, 3, P, 1 << 31, P, P), -1, b"2^31"),
    ("append", (None, 3, None, 3, P, P), -1, b"null"),
    ("append", (P, 3, P, 4, None, P), -1, b"null"),
    ("append", (None, 0, None, 0, None, None), 0, b""),
    ("truncate", (P, P, -1, None, 0, P), -1, b"rows"),
    ("truncate", (P, P, 1, None, 1, P), -1, b"null"),
    ("truncate", (P, None, 1, None, 0, P), -1, b"null"),
    ("truncate", (P, P, 1, P, 1 << 30, P), -1, b"page ids"),
    ("truncate", (None, None, 0, None, 0, None), 0, b""),
    ("fork", (P, P, 8193, 1, P), -1, b"rows"),
    ("fork", (P, None, 1, 1, P), -1, b"null"),
    ("fork", (None, None, 0, 0, None), 0, b""),
    ("compact", (-1, P, P), -1, b"max_moves"),
    ("compact", (1, None, P), -1, b"needed"),
    ("compact", (1, P, P + 4), -1, b"8-byte"),
    ("compact", (1, P, None), -1, b"needed"),
])
def test_entry_points_refuse_bad_lists(call, args, code, msg):
    lib = _lib.lib()
    rc = getattr(lib, "nkv_pages_" + call)(_args(), *args, None)
    assert rc == code and msg in lib.nkv_last_error(), lib.nkv_last_error()
    assert getattr(lib, "nkv_pages_" + call)(None, *args, None) == -1


def test_workspace_bytes():
    f = _lib.lib().nkv_pages_workspace_bytes
    assert f(0) == f(-1) == f((1 << 20) + 1) == 0
    assert f(1000) == 64 + 16 * 8192 + 24 * 1000


@pytest.mark.parametrize("max_moves", [(1 << 20) + 1, (1 << 31) - 1024, (1 << 31) - 1])
def test_compact_refuses_more_moves_than_a_pool_can_have(max_moves):
    """The list's padding is counted in 32 bits, 1024 entries a step."""
    lib = _lib.lib()
    assert lib.nkv_pages_compact(_args(), max_moves, P, P, None) == -1
    assert b"max_moves" in lib.nkv_last_error()


@pytest.fixture
def host_pool(monkeypatch):
    """A PagedSequences over host tensors, whose calls are recorded: (entry point, arguments)."""
    calls = []

    class Lib:
        nkv_pages_workspace_bytes = staticmethod(_lib.lib().nkv_pages_workspace_bytes)

        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    lib = Lib()
    monkeypatch.setattr(_lib, "require_device", lambda *a, **kw: None)
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(_lib, "device_of", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    seqs = pages.PagedSequences(torch.zeros(2, 1, 4, 16, 2, 64, dtype=torch.bfloat16), 3, 2)
    seqs.calls = calls
    return seqs


def test_state_and_pool_cannot_be_set(host_pool):
    """The calls go on with the buffers that the object was made over, so that its views have to."""
    kept = host_pool.state.clone()
    for name in ("state", "kv_cache"):
        with pytest.raises(AttributeError):
            setattr(host_pool, name, getattr(host_pool, name).clone())
    host_pool.state[4] = 9
    assert host_pool.context_lens.tolist() == [9, 0, 0]
    host_pool.state.copy_(kept)
    host_pool.compact()
    name, args = host_pool.calls[-1]
    assert name == "nkv_pages_compact" and struct.unpack("13q", args[0])[5] == \
        host_pool.state.data_ptr() == host_pool.ref_counts.data_ptr()
    assert host_pool.context_lens.tolist() == [0, 0, 0]


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s))])
def test_a_copy_gives_the_kernels_its_own_buffers(host_pool, how):
    calls = host_pool.__dict__.pop("calls")
    host_pool.state[5] = 3
    other = how(host_pool)
    other.compact()
    args = struct.unpack("13q", calls[-1][1][0])
    assert args[0] == other.kv_cache.data_ptr() and args[5] == other.state.data_ptr()
    assert args[11] != struct.unpack("13q", host_pool._args)[11]  # a workspace of its own
    assert (args[5] == host_pool.state.data_ptr()) == (how is copy.copy)
    assert other.context_lens.tolist() == [0, 3, 0]
    assert (other.max_seqs, other.max_blocks, other.block_size) == (3, 2, 16)


def test_buffers_outlive_the_object_where_a_graph_captured_them(host_pool, monkeypatch):
    """A replay writes the plan to the workspace's address, whoever still holds the object."""
    attn = importlib.import_module("nanokv-llm_amd.layers.attention")
    monkeypatch.setattr(attn, "_RETIRED_WS", [])
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    calls = host_pool.__dict__.pop("calls")
    eager, graph = (copy.deepcopy(host_pool) for _ in range(2))
    eager.compact()
    graph.compact()
    capturing[0] = True
    graph.compact()
    graph.compact()
    capturing[0] = False
    args = struct.unpack("13q", calls[-1][1][0])
    del eager
    assert attn._RETIRED_WS == []
    del graph
    (kept,) = attn._RETIRED_WS
    assert [t.data_ptr() for t in kept] == [args[11], args[5]]
    assert attn.release_retired_decode_workspaces() == 1 and attn._RETIRED_WS == []


def test_buffers_are_recorded_on_other_streams_than_their_own(host_pool, monkeypatch):
    """Freed memory goes to its own stream's next allocation at once, so that what runs elsewhere
    has to be known to the allocator: once a stream."""
    recorded = []

    class Seen(torch.Tensor):
        def record_stream(self, stream):
            recorded.append((self.data_ptr(), stream))

    stream = [7]
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: stream[0],
                        raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: f"stream {stream[0]}")
    host_pool._workspace = host_pool._workspace.as_subclass(Seen)
    host_pool._state = host_pool._state.as_subclass(Seen)
    for stream[0] in (7, 8, 8, 7, 9):
        host_pool.compact()
    both = [host_pool._workspace.data_ptr(), host_pool._state.data_ptr()]
    assert recorded == [(p, f"stream {s}") for s in (8, 9) for p in both]


def free_page_listed(p):
    """Two rows share pages; one is cut inside a shared page, so that it takes the lowest free page
    for its copy, and the same call lists that page and the next free one."""
    assert p.append([0], [40]) == [1] and p.fork([0], [1]) == [1]
    free = [x for x, c in enumerate(p.ref.refs) if c == 0]
    assert p.truncate([1], [20], pages=[free[0], free[1], free[0]]) == [1]
    assert p.ref.tables[1][1] == free[0] and p.ref.refs[free[0]] == 1
    held = [x for t in p.ref.tables for x in t if x >= 0]
    assert p.ref.refs == [held.count(x) for x in range(len(p.ref.refs))]
    assert p.append([2], [40]) == [1]  # takes other pages
    assert not set(p.ref.tables[2]) & set(p.ref.tables[1]) - {-1}


class OracleAlone:
    def __init__(self):
        self.ref = PagedSequencesRef(torch.zeros(2, 1, 40, 16, 1, 1, dtype=torch.int64), 8, 6)

    def append(self, rows, counts):
        return self.ref.append(rows, cu=[sum(counts[:i]) for i in range(len(counts) + 1)],
                               n_tokens=sum(counts))[1]

    def fork(self, parents, children):
        return self.ref.fork(parents, children)

    def truncate(self, rows, lens, pages):
        return self.ref.truncate(rows, lens, pages)


def test_a_listed_page_that_was_free_keeps_its_new_row():
    free_page_listed(OracleAlone())
