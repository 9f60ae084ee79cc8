"""lookup_tree (host): drafts are the continuations of earlier occurrences, shared beginnings once."""
from tinferno_b200.model import lookup_tree


def test_continuations_of_the_latest_occurrences():
    text = [7, 8, 1, 2, 3, 7, 8, 1, 9, 7, 8]
    tokens, parents = lookup_tree(text, 3, 3, 64)
    assert tokens == [8, 1, 9, 7, 2, 3] and parents == [-1, 0, 1, 2, 1, 4]


def test_one_token_when_two_do_not_repeat():
    assert lookup_tree([4, 5, 6, 5], 2, 2, 64) == ([5, 6, 5], [-1, 0, 1])
    assert lookup_tree([1, 2, 3], 2, 2, 64) == ([3], [-1])
    assert lookup_tree([1], 2, 2, 64) == ([1], [-1])


def test_room_and_order():
    text = [1, 2, 3, 4, 5, 6, 1, 2, 9, 9, 1, 2]
    for room in range(1, 8):
        tokens, parents = lookup_tree(text, 4, 4, room)
        assert len(tokens) <= room and parents[0] == -1
        assert all(0 <= p < i for i, p in enumerate(parents) if i)
