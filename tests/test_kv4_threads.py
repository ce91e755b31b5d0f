"""A 4-bit cache shared by host threads."""
import copy
import pickle
import random
import sys
import threading

from b200attn.kv4 import KV4Cache, OutOfPages, PageTables


def test_threads_share_the_accounting():
    """Threads that add, fork, extend and free at once lose no page and share none that they
    should not."""
    cache = KV4Cache(1, 1, 40, device="cpu")
    failed, old = [], sys.getswitchinterval()

    def work(seed):
        rng, mine = random.Random(seed), []
        try:
            for _ in range(400):
                try:
                    op = rng.randrange(4)
                    if op == 0 or not mine:
                        mine += cache.add([rng.choice((1, 64, 100)) for _ in range(3)])
                    elif op == 1:
                        mine += cache.fork([rng.choice(mine)])
                    elif op == 2:
                        s = rng.choice(mine)
                        cache.extend([s], [-cache.tables.length(s) % 64 + 64 if
                                           cache.tables._uses[cache.tables.pages(s)[-1]] == 1 else 0])
                    else:
                        cache.free([mine.pop(rng.randrange(len(mine)))])
                except OutOfPages:
                    while mine:
                        cache.free([mine.pop()])
            cache.free(mine)
        except Exception as e:
            failed.append(repr(e))

    try:
        sys.setswitchinterval(1e-6)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(old)
    assert not failed, failed[:3]
    assert sorted(cache.tables._free) == list(range(40)) and not any(cache.tables._uses)


def test_tables_can_be_copied_and_pickled():
    """A copy plans ahead without touching the tables themselves."""
    tables = PageTables(6)
    a = tables.add(100)
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables))):
        other.extend([other.fork(a)], [70])
        assert other.free_pages == 2 and other.pages(a) == [0, 1]
        assert tables.free_pages == 4 and tables.pages(a) == [0, 1]
        assert other.lock is not tables.lock
