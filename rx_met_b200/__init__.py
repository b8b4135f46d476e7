def wait_gave_up() -> bool:
    """Whether a bounded wait inside a kernel of the token mixer has run out on the current device since the process began (the results of that call are not to be used)."""
    from . import _cabi
    return _cabi.wait_gave_up()
