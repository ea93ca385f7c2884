"""Which form of the kernel an attention over pages takes: the rules of akv_paged_attention.cu, .h and .cuh again, for tests that have to reach every form."""
CHUNK, TEAM_CHUNK, MOST_WARPS = 64, 32, 16
ROW = {"fp16": 2, "e4m3": 1, "e2m1": 0.5}           # bytes of a channel


def cdiv(a, b):
    return -(-a // b)


def warps_of(form, D, nt):
    if form == "e2m1" and D == 128 and nt == 1:
        return 16
    return 12 if nt == 1 or D == 64 and (nt == 2 or nt == 3 and form != "fp16") else 8


def step_tokens(form, D, nt):
    row = int(ROW[form] * D)
    return 16 * (1 if row == 256 else 4 if row < 128 and D == 64 and nt <= 2 else 2)


def plan(form, D, B, H, group, T, page, width, sms=148):
    """(tiles of 8 rows, CTAs of a unit's cluster or 0, bytes of the workspace)."""
    rows, heads, table = group * T, B * H, width * page
    eights = cdiv(rows, 8)
    groups = eights if heads * eights * cdiv(table, CHUNK) <= 2 * sms * MOST_WARPS else cdiv(rows, 32)
    nt = cdiv(cdiv(rows, groups), 8)
    warps, chunks, units, team = warps_of(form, D, nt), cdiv(table, TEAM_CHUNK), heads * groups, 8
    while team > 1 and (units * team > sms * 3 // 4 or team // 2 * warps >= 2 * chunks):
        team //= 2
    if units * team > sms or chunks > 8 * warps * team:
        team = 0
    return nt, team, 0 if team else (2 + MOST_WARPS) * sms * 8 * nt * (D + 4) * 4 + 8 * sms


def form_of(form, D, B, H, group, T, page, width, sms=148):
    """(format, channels, tiles, a step lies in one page, by clusters, rows twice in their tile)."""
    nt, team, _ = plan(form, D, B, H, group, T, page, width, sms)
    rows = group * T
    unit = cdiv(rows, cdiv(rows, 8)) if nt == 1 and rows > 8 else rows
    return form, D, nt, step_tokens(form, D, nt) <= page, team > 0, nt == 1 and unit <= 4


def all_forms():
    return {(form, D, nt, one, team, twice) for form in ROW for D in (64, 128) for nt in (1, 2, 3, 4) for one in (True, False) for team in (True, False)
            for twice in ((True, False) if nt == 1 else (False,)) if one or step_tokens(form, D, nt) > 16}


# Tables of 52 (sequence, KV head) pairs: of 3000 tokens a cluster per pair, of 200000 equal runs; (query heads of a KV head, new tokens) of every tile count.
B, H, TABLES, PAGES = 13, 4, (3000, 200000), (16, 64)
ROWS = [(1, 3), (4, 1), (1, 6), (8, 1), (3, 4), (16, 1), (4, 5), (24, 1), (8, 4), (5, 5)]
LENS = (0, 1, 15, 16, 64, 65, 127, 200, 333, 512, 700, 1029, 2950)
