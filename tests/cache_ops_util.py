"""Inputs of the tests of the operators around a long paged cache."""
import torch

BF = torch.bfloat16


def gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(k) for i, k in enumerate(key)) % (1 << 31))


def tables(g, lens, block_size, spare=2, width=None):
    """Tables over pages in a random order, -1 behind a sequence's last page, and the number of pages in all."""
    used = [max(0, -(-n // block_size)) for n in lens]
    total = sum(used) + spare
    perm = torch.randperm(total, generator=g).to(torch.int32)
    out = torch.full((len(lens), width or max(1, max(used))), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        out[b, :u] = perm[at:at + u]
        at += u
    return out, total


def angles(top, rot, theta=500000.0):
    inv = 1.0 / theta ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(top, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def within(got, want, slack):
    """got is want up to slack, NaN where want is NaN."""
    got = got.double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    far = ((got - want).abs() - slack)[~nan]
    assert far.numel() == 0 or float(far.max()) <= 0, f"off by {float(far.max())} more than allowed"


#: place: (lengths in the cache, new tokens, pages to hand out, of them gone, rows, block_size, width of the tables)
PLACES = {
    "one": ([0], [1], 3, 0, 1, 16, 4),
    "decode": ([5, 16, 31, 0, 48], [1, 1, 1, 1, 1], 9, 2, 8, 16, 5),
    "verify_padded": ([250, 256, 700], [7, 7, 7], 6, 1, 32, 256, 4),
    "prompts_ragged": ([0, 3, 64, 0, 130], [70, 61, 1, 0, 127], 12, 0, 300, 64, 5),
    "pages_short": ([15, 16, 16, 14], [1, 1, 2, 2], 1, 0, 9, 16, 3),          # the second takes the only page, the third waits; the fourth needs none... of the third's
    "rows_short": ([0, 0, 5, 0], [4, 5, 0, 1], 9, 0, 8, 16, 2),                # the second has no room, the third asks for none, the fourth stays behind it
    "used_up": ([0, 3], [1, 1], 4, 7, 4, 16, 2),                               # more gone than there were
    "used_negative": ([0], [20], 4, -3, 20, 16, 2),
    "bad_lengths": ([-1, 4, 10, 30], [1, -2, 100, 2], 9, 0, 64, 16, 2),        # negative, negative, past the table, just within it
    "huge": ([2147483647, 0, 5], [2147483647, 2147483647, 3], 4, 0, 6, 16, 2),
    "nothing": ([0, 7], [0, 0], 0, 0, 3, 16, 2),
    "no_free_list": ([0, 7], [1, 3], 0, 0, 6, 16, 2),
}


def place_case(name):
    ctx, new, n_free, used, rows, block_size, width = PLACES[name]
    lens = [min(max(c, 0), width * block_size) for c in ctx]
    table, total = tables(gen(len(ctx), rows), lens, block_size, spare=n_free, width=width)
    left = [p for p in range(total) if p not in set(table.flatten().tolist())]
    return ctx, new, table, left[:n_free], used, rows, block_size, total
