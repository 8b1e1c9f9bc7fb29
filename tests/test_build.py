"""When the library counts as up to date.  The compiler's place is taken by a stand-in that writes empty files."""
import os

import pytest

from vqa_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """One source that was built an hour ago, by a recipe that is older still; the commands run since."""
    ran = []

    class Compile:
        def __init__(self, cmd):
            ran.append(cmd)
            open(cmd[cmd.index('-o') + 1], 'w').close()

        def wait(self):
            return 0
    for name in ('a.hip', 'a.h', 'recipe.py', 'a.o', 'lib.so'):
        (tmp_path / name).touch()
    now = os.path.getmtime(tmp_path / 'lib.so')
    for i, name in enumerate(('a.hip', 'a.h', 'recipe.py', 'a.o', 'lib.so')):
        os.utime(tmp_path / name, (now - 3600 + i, now - 3600 + i))
    for k, v in dict(CSRC=str(tmp_path), OUT=str(tmp_path / 'lib.so'), SOURCES=['a.hip'], HEADERS=['a.h'],
                     __file__=str(tmp_path / 'recipe.py')).items():
        monkeypatch.setattr(build, k, v)
    monkeypatch.setattr(build.subprocess, 'Popen', Compile)
    monkeypatch.setattr(build.subprocess, 'check_call', lambda cmd: Compile(cmd).wait())
    return tmp_path, ran


def test_nothing_is_built_twice(tree):
    build.build(verbose=False)
    assert tree[1] == []


@pytest.mark.parametrize('changed', ['a.hip', 'a.h', 'recipe.py'])
def test_a_change_to_a_source_a_header_or_the_recipe_builds_again(tree, changed):
    """(The compiler's flags stand in the recipe.)"""
    path, ran = tree
    os.utime(path / changed)
    build.build(verbose=False)
    assert len(ran) == 2                                       # compiled and linked
    del ran[:]
    build.build(verbose=False)
    assert ran == []


def test_objects_need_not_be_there(tree):
    os.remove(tree[0] / 'a.o')
    build.build(verbose=False)
    assert tree[1] == []
