"""Freeing a request costs what its blocks cost where nothing is shared."""

from mini_infra_b200.core import KVCacheManager


class Counted(dict):
    looked_up = 0

    def pop(self, *args):
        Counted.looked_up += 1
        return super().pop(*args)


def test_sharing_is_looked_up_only_where_there_is_some():
    m = KVCacheManager(4, 40)
    m._sharers = Counted()
    assert m.allocate_slots(0, 50) and m.allocate_slots(1, 10)
    m.free(1)
    assert Counted.looked_up == 0 and m.num_used_blocks == 13
    copies = m.fork(0, 2)
    assert len(copies) == 1 and m.num_used_blocks == 14
    m.free(0)
    assert Counted.looked_up == 13 and m.num_used_blocks == 13 and not m._sharers
    m.free(2)
    assert Counted.looked_up == 13 and m.num_used_blocks == 0
