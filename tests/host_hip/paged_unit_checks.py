"""The units that rows of heads move in (ge_op_rotate_heads, ge_op_paged_append) by head dim, part, strides and
addresses together, on the host HIP runtime (host_hip.cpp). Run by tests/test_paged_units_host.py in a process
of its own, whose GE_LIBRARY is the library's objects over that runtime."""
import pytest

from paged_checks import BF16, F16, F32, Launches, append, ctx, memory, rotate, table, unit_of  # noqa: F401 (fixtures)


def unit(head_dim, dims, in_size, strides, addresses):
    """The largest unit that the header's rule allows and whose two halves of a head fit a wave's lanes. strides and
    addresses: (elements or bytes, whether of the input) of every operand."""
    for u in (8, 4, 2):
        def piece(of_input):  # elements of an access, up to 16 bytes
            return min(u, 16 // in_size if of_input else 8)
        if head_dim % (2 * u) or dims // 2 % u or head_dim // 2 // u > 64:
            continue
        if all(s % piece(i) == 0 for s, i in strides) and all(a % (piece(i) * (in_size if i else 2)) == 0 for a, i in addresses):
            return u
    return 1


@pytest.mark.parametrize("in_type", [F16, F32])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 258, 264, 320, 384, 504, 512])
@pytest.mark.parametrize("moved", [0, 2, 4, 8, 16])
def test_units_of_long_heads_at_any_address(ctx, memory, in_type, head_dim, moved):
    """From head dim 258 on a wave's lanes hold no head in units of 2: what an address does not let move in units
    of 4 moves in units of 1."""
    size = 4 if in_type == F32 else 2
    if moved % size:
        moved += 2
    for dims in (0, head_dim // 2 // 2 * 2, 16):
        handle = ctx.rotary_create(dims, 1e4) if dims else None
        for name in ("q", "k", "q_out", "k_out"):
            place = {n: memory + (16384 if n.endswith("out") else 0) for n in ("q", "k", "q_out", "k_out")}
            place[name] += moved
            width = [4 * head_dim, 2 * head_dim]
            want = unit(head_dim, dims, size, [(w, i) for w in width for i in (True, False)], [(place[n], not n.endswith("out")) for n in place])
            with Launches() as got:
                rotate(ctx, memory, handle, dict(head_dim=head_dim, in_type=in_type), **place)
            assert [unit_of(n) for n in got.names] == [want], (name, dims)
        if handle:
            ctx.rotary_destroy(handle)


@pytest.mark.parametrize("in_type", [F16, F32])
@pytest.mark.parametrize("head_dim", [128, 264, 512])
@pytest.mark.parametrize("moved", [4, 8])
def test_units_of_an_append_at_any_address(ctx, memory, table, in_type, head_dim, moved):
    size = 4 if in_type == F32 else 2
    for name in ("q", "k", "v", "q_out", "k_pages", "v_pages"):
        place = {n: memory + (16384 if n in ("q_out", "k_pages", "v_pages") else 0) for n in ("q", "k", "v", "q_out", "k_pages", "v_pages")}
        place[name] += moved
        want = unit(head_dim, 0, size, [], [(p, n in ("q", "k", "v")) for n, p in place.items()])
        with Launches() as got:
            append(ctx, memory, None, table, [(0, 3, 0, 50)], dict(head_dim=head_dim, in_type=in_type, type=F16), **place)
        assert [unit_of(n) for n in got.names] == [want], name


@pytest.mark.parametrize("stride", [2050, 2052, 2056])
def test_strides_and_addresses_together(ctx, memory, stride):
    """A stride in units of 2, 4 or 8 and an address in units of 2, of heads of 512."""
    for moved in (0, 4, 8):
        want = unit(512, 0, 2, [(stride, True)], [(memory + moved, True)])
        with Launches() as got:
            rotate(ctx, memory, None, dict(head_dim=512, q_stride=stride, type=BF16, in_type=BF16), q=memory + moved, q_out=memory + 16384,
                   k_out=memory + 16384, positions=None)
        assert [unit_of(n) for n in got.names] == [want]
