def test_the_entry_compiles_where_a_library_is_there(monkeypatch, lib):
    """A change of the compiler's flags leaves every file's time as it was."""
    import __graft_entry__
    from artdeco_amd import _lib, build
    asked = []
    monkeypatch.setattr(build, "build", lambda **kw: (asked.append(kw), _lib.LIB_PATH)[1])
    __graft_entry__.build()
    assert asked and asked[0]["force"]
