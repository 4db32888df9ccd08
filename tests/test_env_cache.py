"""The table of OpEnvs under several threads, without a GPU."""
import sys
import threading


def test_threads_that_push_each_others_entries_out():
    """More signatures than the table holds, from several threads at once: an entry that is found may be pushed
    out by another thread the next moment, which is no error of the thread that found it."""
    from raf_amd import op

    class Small(op._EnvCache):
        capacity = 3

    table, errors, start = Small(), [], threading.Barrier(4)

    def work(k):
        start.wait()
        try:
            for i in range(40_000):
                key = (i * (k + 1)) % 7
                env = table.get(key)
                if env is None:
                    env = table[key] = (key,)
                assert env == (key,)
        except BaseException as e:  # noqa: BLE001
            errors.append(repr(e))

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sys.setswitchinterval(interval)
    assert not errors
    assert len(table) <= 3 + 4  # each thread may be about to drop one


def test_least_recently_used_entry_goes_first():
    from raf_amd import op

    class Small(op._EnvCache):
        capacity = 2

    table = Small()
    table["a"], table["b"] = 1, 2
    assert table.get("a") == 1 and table.get("c") is None and table.get("c", 5) == 5
    table["c"] = 3
    assert list(table) == ["a", "c"]
    table["a"] = 4
    table["d"] = 6
    assert list(table) == ["a", "d"] and table.get("a") == 4
