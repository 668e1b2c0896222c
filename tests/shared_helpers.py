"""Attention over a paged cache in 64 bits, token by token, and inputs whose groups share their first pages."""

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def made(groups, *, num_q=4, num_kv=2, dim=64, page=16, dtype=torch.bfloat16, seed=0, padding=(), own_pages_of_shared=False,
         tokens_of=None, device="cuda"):
    """``groups``: (shared length, [keys each member has behind it]).  ``padding``: tokens that are none.  ``tokens_of``: tokens
    a member has in the step (its last ones; default 1).  ``own_pages_of_shared``: members hold pages of their own for the page in
    which the shared keys end (with the same keys up to there)."""
    gen = torch.Generator().manual_seed(seed)
    tables, positions, starts, rows, pages, copies = [], [], [0], [], 0, []
    for shared, members in groups:
        whole, rest = divmod(shared, page)
        common = list(range(pages, pages + whole))
        pages += whole
        for i, own in enumerate(members):
            table = list(common)
            more = -(-(rest + max(own, 0)) // page)
            mine = list(range(pages, pages + more))
            pages += more
            if rest and mine:
                copies.append((mine[0], rest, (len(starts) - 1, i)))
            tables.append(table + mine)
            count = tokens_of or 1
            for t in range(count):
                positions.append(shared + own - count + t)
                rows.append(len(tables) - 1)
        starts.append(len(positions))
    place = torch.randperm(pages + 3, generator=gen)
    width = max([len(t) for t in tables] + [1]) + 1
    table = torch.full((len(tables), width), -1, dtype=torch.int32)
    for r, t in enumerate(tables):
        table[r, :len(t)] = place[torch.tensor(t, dtype=torch.long)].to(torch.int32)
    tokens = len(positions)
    keys, values = (torch.randn(pages + 3, num_kv, page, dim, generator=gen).to(dtype) for _ in range(2))
    first = {}
    for at, rest, (group, i) in copies:                               # the same keys in every member's own copy of the page
        if group not in first:
            first[group] = place[at]
        else:
            keys[place[at], :, :rest], values[place[at], :, :rest] = keys[first[group], :, :rest], values[first[group], :, :rest]
    positions, rows = torch.tensor(positions, dtype=torch.int32), torch.tensor(rows, dtype=torch.int32)
    for t in padding:
        positions[t], rows[t] = (-1, rows[t]) if t % 2 else (positions[t], -1)
    state = dict(q=torch.randn(tokens, num_q * dim, generator=gen).to(dtype), key_cache=keys, value_cache=values, block_tables=table,
                 token_row=rows, positions=positions, group_starts=torch.tensor(starts, dtype=torch.int32),
                 shared_lens=torch.tensor([s for s, _ in groups], dtype=torch.int32))
    return {name: t.to(device) for name, t in state.items()}, dict(num_q=num_q, num_kv=num_kv, head_dim=dim, scale=dim**-0.5)


def plain_attention(s, num_q, num_kv, head_dim, scale):
    """(values, bounds) in 64 bits.  A score is a float32 sum of head_dim products, off by at most (head_dim + 4) 2^-23 of the
    products' sizes (scaling and the exponent's rounding among them); a weight is off by that share of itself and by 2^-20 (the
    exponential and the joining factors of the pieces, all float32), for bfloat16 by 2^-8 (rounded for the product) too, the sums over
    n keys by n 2^-23; the result is rounded once."""
    q, keys, values = s["q"].double(), s["key_cache"].double(), s["value_cache"].double()
    tokens, page = q.shape[0], keys.shape[2]
    out = torch.zeros(tokens, num_q, head_dim, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    half = HALF_STEP[s["q"].dtype]
    for t in range(tokens):
        row, position = int(s["token_row"][t]), int(s["positions"][t])
        if row < 0 or position < 0:
            continue
        where = torch.arange(min(position + 1, s["block_tables"].shape[1] * page), device=q.device)
        pages = s["block_tables"][row, where // page].long()
        seen = (pages >= 0) & (pages < keys.shape[0])
        where, pages = where[seen], pages[seen]
        k, v = keys[pages, :, where % page].transpose(0, 1), values[pages, :, where % page].transpose(0, 1)    # [kv, keys, size]
        mine = q[t].view(num_kv, num_q // num_kv, head_dim)
        weights = torch.softmax(mine @ k.transpose(1, 2) * scale, dim=-1)
        off = (head_dim + 4) * 2.0**-23 * (mine.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale
        share = 2 * off + 2.0**-20 + where.numel() * 2.0**-23 + (half if half > 2.0**-20 else 0.0)
        out[t] = (weights @ v).reshape(num_q, head_dim)
        bound[t] = (share * (weights @ v.abs())).reshape(num_q, head_dim)
    bound += half * (out.abs() + bound)
    return out.reshape(tokens, -1), bound.reshape(tokens, -1)


def check_attention(got, s, **sizes):
    want, bound = plain_attention(s, **sizes)
    assert got.shape == want.shape and torch.isfinite(got).all()
    off = (got.double() - want).abs() - bound
    assert off.numel() == 0 or off.max().item() <= 0.0, f"{off.max().item():.3g} beyond the bound"
