"""Numbers and places of pages, on the host: what is taken, given back and gathered into pools of other sizes."""
import random
from importlib import import_module

import numpy as np
import pytest


@pytest.mark.parametrize("seed", range(20))
def test_pages_keep_their_numbers_and_their_contents_wherever_they_are_moved(seed):
    Pages, rng = import_module("turboquant-pytorch_amd.paged_cache")._Pages, random.Random(seed)
    size = rng.randint(1, 30)
    pages, pool, held, serial = Pages(size), [None] * size, {}, 0        # held: number -> (what was written, how many hold it)
    for _ in range(300):
        what = rng.choice(("take", "take", "share", "drop", "drop", "gather"))
        if what == "take" and pages.free:
            number = pages.take()
            assert number not in held and number == min([number] + pages.free)
            serial += 1
            pool[int(pages.lie(np.array([number]))[0])] = serial
            held[number] = (serial, 1)
        elif what == "share" and held:
            number = rng.choice(sorted(held))
            pages.held[number] += 1
            held[number] = (held[number][0], held[number][1] + 1)
        elif what == "drop" and held:
            number = rng.choice(sorted(held))
            value, n = held.pop(number)
            assert pages.drop(number) == (n == 1)
            if n > 1:
                held[number] = (value, n - 1)
        elif what == "gather" and rng.random() < 0.3:
            numbers = pages.numbers()
            assert numbers.tolist() == sorted(held)
            size = max(1, len(held)) + rng.choice((0, 0, 1, rng.randint(0, 40)))
            pool = [pool[i] for i in pages.lie(numbers)] + [None] * (size - len(numbers))
            pages = pages.gathered(numbers, size)
        assert len(pages.free) + len(held) == size == len(pool) and not set(pages.free) & set(held)
        places = pages.lie(np.array(sorted(held) + pages.free, dtype=np.int64)).tolist()
        assert sorted(places) == list(range(size))
        assert [pool[i] for i in places[:len(held)]] == [held[n][0] for n in sorted(held)]
        assert all(pages.held[n] == held[n][1] for n in held) and sum(map(bool, pages.held)) == len(held)
