"""Reordered requests of the paged cache by the rule, one row and block after another."""


def reorder(parents, lens, tables, free, num_free, block, num_blocks):
    """(tables, lengths, stack, its size, sources, targets) as lists."""
    rows, width = len(lens), len(tables[0]) if len(tables) else 0
    lens = [max(n, 0) for n in lens]
    used = [min(-(-n // block), width) for n in lens]
    stack = list(free[:max(min(num_free, len(free), num_blocks), 0)])
    real = [p if 0 <= p < rows else None for p in parents]
    held = set()
    for p in real:
        if p is not None:
            held.update(tables[p][:used[p]])
    freed = {b for r in range(rows) for b in tables[r][:used[r]] if 0 <= b < num_blocks} - held
    stack += sorted(freed)
    out, out_lens, sources, targets, seen, missing = [], [], [], [], set(), 0
    for p in real:
        n = 0 if p is None else lens[p]
        row = [] if p is None else list(tables[p][:used[p]])
        row += [-1] * (width - len(row))
        source = target = -1
        at = n // block
        if p is not None and n % block and at < width and p in seen and 0 <= row[at] < num_blocks:
            source = row[at]
            if stack:
                target = stack.pop()
            else:
                missing += 1
            row[at] = target
        seen.add(p)
        out.append(row)
        out_lens.append(n)
        sources.append(source)
        targets.append(target)
    left = len(stack) - missing
    return out, out_lens, stack + [-1] * (num_blocks - len(stack)), left, sources, targets
