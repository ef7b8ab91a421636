"""Calls of paged_append and paged_read in 8 bits whose workgroups walk over several heads, which neither number of heads
divides among.  `threads` of the append's workgroups; `append` and `read`: the heads of a walk."""

NEW = [1037, 900, 1, 1062]
CONTEXT = [1037, 907, 301, 1100]  # none, 7, 300 and 38 older tokens
LONG = [3037, 2900, 1, 3062]
LONG_CONTEXT = [3040, 2907, 301, 3062]

CASES = {
    "turned_16": dict(new=NEW, context=CONTEXT, d=128, page=32, block=16, hq=39, threads=256, append=8, read=4),
    "turned_64": dict(new=NEW, context=CONTEXT, d=128, page=64, block=64, hq=39, threads=1024, append=8, read=4),
    "turned_128": dict(new=NEW, context=CONTEXT, d=128, page=128, block=128, hq=39, threads=1024, append=5, read=4),
    "turned_narrow": dict(new=NEW, context=CONTEXT, d=64, page=96, block=48, hq=39, threads=512, append=7, read=2),
    "plain_16": dict(new=NEW, context=CONTEXT, d=128, page=16, block=16, hq=0, threads=256, append=4, read=4),
    "plain_narrow": dict(new=LONG, context=LONG_CONTEXT, d=64, page=64, block=64, hq=0, threads=256, append=3, read=7),
    "plain_64": dict(new=LONG, context=LONG_CONTEXT, d=128, page=64, block=64, hq=0, threads=256, append=3, read=8),
}
HEADS = 13  # of k and v
