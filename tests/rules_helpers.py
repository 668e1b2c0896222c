"""Rules on logits in 64 bits, and the bound on what float32 arithmetic may be off by."""

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def plain_rules(logits, slots, penalties, lengths, history, bias_tokens=None, bias_values=None, masks=None, mask_rows=None):
    """(values, bounds) in 64 bits, row by row and token by token of what the rules name.

    The bound: a value passes through at most five float32 operations (penalty, product, two differences, sum; a token
    named n times adds n - 1 sums), each off by at most half a step of a number no larger than what all of them add up to
    in size, and one rounding to the logits' type."""
    wide = torch.float64
    out, bound = logits.to(wide).clone(), torch.zeros(logits.shape, dtype=wide)
    rows, vocab = logits.shape
    for r in range(rows):
        slot = int(slots[r])
        if not 0 <= slot < history.shape[0]:
            continue
        repetition, presence, frequency = (float(p) for p in penalties[slot])
        total = min(max(int(lengths[slot, 0]), 0), history.shape[1])
        prompt = min(max(int(lengths[slot, 1]), 0), total)
        counts, seen = {}, set()
        for i in range(total):
            token = int(history[slot, i])
            if 0 <= token < vocab:
                seen.add(token)
                if i >= prompt:
                    counts[token] = counts.get(token, 0) + 1
        size, steps = {}, {}
        for token in seen:
            x = out[r, token].item()
            x = x / repetition if x > 0 else x * repetition
            size[token], steps[token] = abs(x), 4
            if token in counts:
                x = x - frequency * counts[token] - presence
                size[token] += abs(frequency) * counts[token] + abs(presence)
            out[r, token] = x
        for i in range(0 if bias_tokens is None else bias_tokens.shape[1]):
            token = int(bias_tokens[slot, i])
            if 0 <= token < vocab:
                size[token] = size.get(token, abs(out[r, token].item())) + abs(float(bias_values[slot, i]))
                steps[token] = steps.get(token, 0) + 1
                out[r, token] += float(bias_values[slot, i])
        for token in size:
            bound[r, token] = steps[token] * HALF_STEP[torch.float32] * size[token] * (1 + 2.0**-20)
        if masks is not None and 0 <= int(mask_rows[slot]) < masks.shape[0]:
            for token in range(vocab):
                if not (int(masks[int(mask_rows[slot]), token // 32]) >> (token % 32)) & 1:
                    out[r, token], bound[r, token] = float("-inf"), 0.0
    most = torch.finfo(logits.dtype).max * (1 + HALF_STEP[logits.dtype] / 2)          # from here on a number rounds to infinity
    out = torch.where(out.abs() >= most, out.sign() * float("inf"), out)
    if logits.dtype != torch.float32:
        bound = bound + HALF_STEP[logits.dtype] * (out.abs() + bound).nan_to_num(posinf=0.0)
    return out, bound


def check_rules(got, logits, **rules):
    want, bound = plain_rules(logits.cpu(), **{name: None if t is None else t.cpu() for name, t in rules.items()})
    got = got.cpu().to(torch.float64)
    whole = torch.isfinite(want)
    assert torch.equal(got[~whole], want[~whole]) or torch.equal(torch.nan_to_num(got[~whole]), torch.nan_to_num(want[~whole]))
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got[whole] - want[whole]).abs() - bound[whole]
    assert off.numel() == 0 or off.max().item() <= 0.0, f"off by {off.max().item():.3g} beyond the bound"
