"""Rotary positions' tables, which are shared by contents, without a GPU."""

import threading

from aegaeon_amd import ops


class Table:
    pass


def test_threads_that_make_equal_tables_at_once_share_one(monkeypatch):
    """A table that a stream may be reading is never replaced: the one that is kept is the
    one that every thread was given."""
    monkeypatch.setattr(ops, "_turn_tables", {})
    both, given = threading.Barrier(2, timeout=20), []

    def make():
        both.wait()     # each has found none before either keeps its own
        return Table()

    threads = [threading.Thread(target=lambda: given.append(ops._turn_table((0, b"x"), make)))
               for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert len(given) == 2 and given[0] is given[1]
    assert ops._turn_table((0, b"x"), make) is given[0]
