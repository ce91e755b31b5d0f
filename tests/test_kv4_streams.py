"""A 4-bit cache shared by streams: a page that one stream's queued work still
reads is taken for another's only behind that work."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import b200attn
from b200attn.kv4 import KV4Cache
from test_kv4 import D, i32, values


class FakeStream:
    """A stream as its queue: what was put into it, in order."""
    def __init__(self, handle):
        self.cuda_stream, self.queue = handle, []

    def wait_event(self, event):
        self.queue.append(("wait", event.stream, event.at))


class FakeEvent:
    def record(self, stream):
        self.stream, self.at = stream, len(stream.queue)  # behind everything queued so far


@pytest.fixture
def fake_gpu(monkeypatch):
    """A cache whose pool claims to be on a GPU, and the switch for the current stream."""
    now = SimpleNamespace(stream=FakeStream(0), capturing=False)
    monkeypatch.setattr(torch.cuda, "Event", FakeEvent)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now.stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capturing)
    cache = KV4Cache(1, 1, 4, device="cpu")
    cache.pool = SimpleNamespace(is_cuda=True, device="cuda:0")

    def copy(pool, src, dst):
        now.stream.queue.append(("copy", list(src), list(dst)))
    monkeypatch.setattr(b200attn, "kv4_copy_pages", copy)
    return cache, now


def behind(stream, other, at):
    """Whether `stream` has been made to wait for the first `at` entries of `other`."""
    return any(e[0] == "wait" and e[1] is other and e[2] >= at for e in stream.queue)


@pytest.mark.parametrize("how", ["add", "extend", "compact"])
def test_freed_pages_are_taken_behind_the_work_that_reads_them(fake_gpu, how):
    cache, now = fake_gpu
    one, two = FakeStream(1), FakeStream(2)
    now.stream = two
    other, = cache.add([64])
    now.stream = one
    a, = cache.add([64])
    b, = cache.add([64])
    fork, = cache.fork([other])
    assert cache.tables.pages(b) == [2]
    one.queue.append("reads of a")
    cache.free([a])
    now.stream = two
    if how == "add":
        cache.add([128])
    elif how == "extend":
        cache.extend([other], [1])
    else:
        assert cache.compact() == 1
        assert two.queue[-1][0] == "copy"  # the wait is in front of it
        two.queue.pop()
    assert behind(two, one, one.queue.index("reads of a") + 1)


def test_copied_pages_are_taken_behind_the_copies(fake_gpu):
    """Stream one copies a page that two forks shared, then the one that kept it is freed on
    stream two: a third stream takes it behind the copy."""
    cache, now = fake_gpu
    one, two, three = (FakeStream(i) for i in (1, 2, 3))
    now.stream = two
    kept, = cache.add([10])
    fork, = cache.fork([kept])
    now.stream = one
    cache.extend([fork], [5])
    copied = one.queue.index(("copy", [0], [1])) + 1
    now.stream = two
    cache.free([kept])
    now.stream = three
    assert cache.tables.pages(cache.add([64])[0]) == [0]
    assert behind(three, one, copied)


def test_marks_do_not_grow_and_captures_have_none(fake_gpu):
    cache, now = fake_gpu
    one = FakeStream(1)
    now.stream = one
    for _ in range(20):
        cache.free(cache.add([64]))
    waits = [e for e in one.queue if e[0] == "wait"]
    assert len(waits) <= 20
    one.queue.clear()
    now.capturing = True
    cache.free(cache.add([64]))
    assert one.queue == []


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["free", "extend"])
def test_a_recycled_page_keeps_its_old_readers_values(cuda, how):
    """A slow stream reads a sequence and frees it (or copies a shared page that then is
    freed); at once another stream takes the page and stores other tokens into it."""
    g = torch.Generator().manual_seed(7)
    cache = KV4Cache(1, 2, 2, cuda)
    old, new = (torch.randn(1, 2, 50, D, generator=g).bfloat16() for _ in range(2))
    a, = cache.add([50])
    view = cache.view([a])
    old_dev, new_dev = old.to(cuda), new.to(cuda)
    lengths = i32(cuda, 50)
    view.store(0, old_dev, old_dev)
    slow, fast = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    if how == "free":
        with torch.cuda.stream(slow):
            torch.cuda._sleep(100_000_000)  # some 50 ms
            got = view.load(0, lengths)
            cache.free([a])
    else:
        fork, = cache.fork([a])
        with torch.cuda.stream(slow):
            torch.cuda._sleep(100_000_000)
            cache.extend([fork], [1])       # queues the copy of the shared page
        cache.free([a])
    with torch.cuda.stream(fast):
        b, = cache.add([50])
        taken = cache.view([b])
        taken.store(0, new_dev, new_dev)
    torch.cuda.synchronize()
    assert cache.tables.pages(b) == [0]
    if how == "extend":
        got = cache.view([fork]).load(0, lengths)
    assert torch.equal(got[0][:, :, :50].cpu().double(), values(old))
    assert torch.equal(taken.load(0, lengths)[0].cpu().double(), values(new))
