"""The paged decode where every wave walks several tiles (GPU): tiles loading
while others are computed, rows that begin and end inside a share, running
maxima that move, idle and bad sequences in between."""

import pytest
import torch

from paged_math import assert_within, decode64, pages_for
from refinekv import PagedCache, paged_decode

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _share(lengths, heads, dim):
    """Tiles of 32 tokens that each of the kernel's waves gets at least."""
    tiles = heads * sum(max(1, -(-n // 32)) for n in lengths)
    units = torch.cuda.get_device_properties(0).multi_processor_count
    return tiles // (units * 4 * (2 if dim < 64 else 1))


def _case(lengths, page, heads, group, dim, dtype, seed):
    """Every 150 tokens a key along a query of its head, each longer than the
    one before, so that a row's maximum moves again and again."""
    gen = torch.Generator().manual_seed(seed)
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen)
    query = torch.randn(len(lengths), heads * group, dim, generator=gen).to(dtype)
    for b, n in enumerate(lengths):
        for i, t in enumerate(range(b % 40, n, 150)):
            toward = query[b].view(heads, group, dim)[:, i % group].float()
            at = int(table[b, t // page]), slice(None), t % page
            keys[at] = (toward * 0.2 * (i % 7 + 1)).to(dtype)
    return query, keys, values, table, torch.tensor(lengths, dtype=torch.int32)


def _ragged(count, low, high, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(low, high, (count,), generator=gen).tolist()


@pytest.mark.parametrize("dim,group,page,dtype,scale", [
    (32, 3, 16, BF16, 2), (64, 4, 16, F16, 1), (64, 1, 32, BF16, 1), (96, 2, 64, BF16, 1),
    (128, 4, 16, BF16, 1), (128, 7, 64, F16, 1), (160, 5, 32, F16, 1), (192, 2, 16, BF16, 1),
    (224, 3, 128, F16, 1), (256, 8, 256, BF16, 1), (256, 1, 16, F16, 1),
])
def test_shares_of_several_tiles(dim, group, page, dtype, scale):
    """Long rows, cut into shares of an odd or even number of tiles (and the
    first waves one more); short rows, several of them in a share."""
    heads = 8
    for low, high, count in ((300, 1900, 24 * scale), (1, 100, 330 * scale), (900, 1000, 25 * scale)):
        lengths = _ragged(count, low, high, dim + count)
        lengths[3] = lengths[-2] = 0
        assert _share(lengths, heads, dim) >= 4
        case = _case(lengths, page, heads, group, dim, dtype, dim + high)
        query, *parts = (t.cuda() for t in case)
        got = paged_decode(query, PagedCache(*parts), backend="hip")
        want, room = decode64(*case, dim ** -0.5)
        assert_within(got, want, room, f"{low}..{high}")


def test_shares_of_every_small_size():
    """1 to 9 tiles a wave, to the tile: the loop's two buffers end on either."""
    heads, dim, page = 8, 64, 16
    units = torch.cuda.get_device_properties(0).multi_processor_count * 4
    for share in range(1, 10):
        for extra in (0, 1):
            # two sequences, whole tiles but for the last ones
            tiles = units * share // heads + extra
            lengths = [tiles // 3 * 32 - 5, (tiles - tiles // 3) * 32 - 31]
            case = _case(lengths, page, heads, 1, dim, BF16, share)
            query, *parts = (t.cuda() for t in case)
            got = paged_decode(query, PagedCache(*parts), backend="hip")
            want, room = decode64(*case, dim ** -0.5)
            assert_within(got, want, room, f"{share} tiles, {extra} more")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_bad_and_idle_sequences_inside_shares(dtype):
    """Sequences with a page outside the cache or a length past their table,
    idle and negative ones, each beside sound ones: only their own rows are NaN
    or zero."""
    heads, group, dim, page = 8, 2, 128, 16
    lengths = _ragged(330, 1, 100, 9)
    query, keys, values, table, lens = _case(lengths, page, heads, group, dim, dtype, 5)
    for b in range(0, 330, 11):
        table[b, (lengths[b] - 1) // page // 2] = (-1, keys.shape[0], -2 ** 31, 2 ** 31 - 1)[b % 4]
        lens[b + 1] = table.shape[1] * page + 1
        lens[b + 2] = 2 ** 31 - 1
        lens[b + 3] = 0
        lens[b + 4] = -5 - b
    assert _share(lengths, heads, dim) >= 4
    case = (query, keys, values, table, lens)
    got = paged_decode(query.cuda(), PagedCache(*(t.cuda() for t in case[1:])), backend="hip")
    want, room = decode64(*case, dim ** -0.5)
    assert want.isnan().any(-1).any(-1).sum() == 90 and (want == 0).all(-1).all(-1).sum() == 60
    assert_within(got, want, room)


def test_scores_of_plus_infinity_make_their_row_nan():
    """One token's score of +inf: the softmax's inf / inf, in its rows alone,
    in whole rows, in rows of several waves and of several workgroups."""
    heads, group, dim, page = 2, 2, 64, 16
    for lengths in ([20, 40, 33], [9000, 70, 12]):
        query, keys, values, table, lens = _case(lengths, page, heads, group, dim, BF16, 6)
        clean = (query.clone(), keys.clone(), values, table, lens)
        keys[int(table[0, 1]), 1, 2, 0] = float("inf")   # sequence 0, KV head 1, token 18
        query[0, 2, 0], query[0, 3, 0] = 1.0, -1.0       # its rows: +inf, and -inf
        clean[0][0, 2:4] = query[0, 2:4]
        got = paged_decode(query.cuda(), PagedCache(*(t.cuda() for t in (keys, values, table, lens))),
                           backend="hip").cpu()
        want, room = decode64(*clean, dim ** -0.5)
        assert got[0, 2].isnan().all()
        # -inf: as if the token were not there
        take = table[0, :-(-lengths[0] // page)].long()
        k, v = (t[take, 1].reshape(-1, dim)[:lengths[0]].double() for t in (clean[1], values))
        keep = torch.arange(lengths[0]) != 18
        want[0, 3] = torch.softmax(query[0, 3].double() @ k[keep].T * dim ** -0.5, -1) @ v[keep]
        sound = torch.ones(got.shape[:2], dtype=torch.bool)
        sound[0, 2] = False
        assert_within(got[sound], want[sound], room[sound])
