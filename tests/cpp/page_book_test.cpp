// The bookkeeping of a cache's pages (csrc/page_book.h), against sequences that are kept as plain lists of tokens.  "Device
// memory" is an array of pages and a copy of the words here; moves and changes are carried out on it as the kernels would.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>

#include "../../fyusenet_amd/csrc/page_book.h"

using fynhip::PageBook;

#define CHECK(x)                                                    \
    do {                                                            \
        if (!(x)) {                                                 \
            fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x); \
            exit(1);                                                \
        }                                                           \
    } while (0)

struct Model {
    int pages, sequences, page_tokens;
    PageBook book;
    std::vector<std::vector<int>> want;   // tokens of each sequence
    std::vector<int> pool;                // [page][token]
    std::vector<int> words;
    int next = 1;

    Model(int p, int s, int t, int most) : pages(p), sequences(s), page_tokens(t), book(p, s, t, most), want(s), pool((size_t)p * t, -1), words(book.words.size(), 0) {}

    void moved(const PageBook::Moves& m) {
        std::set<int> from, to;
        for (auto& x : m) { from.insert(x.first); CHECK(to.insert(x.second).second); }
        for (int x : to) CHECK(!from.count(x));
        for (auto& x : m)
            for (int i = 0; i < page_tokens; i++) pool[(size_t)x.second * page_tokens + i] = pool[(size_t)x.first * page_tokens + i];
    }
    void flush() {
        for (auto& c : book.changes())
            for (size_t i = c.first; i < c.second; i++) words[i] = book.words[i];
        book.changes_taken();
    }
    void extend(const std::vector<int>& seqs, const std::vector<int>& counts) {
        moved(book.extend((int)seqs.size(), seqs.data(), counts.data()));
        flush();
        // the rows of the batch, as the kernels find them
        const int n = words[book.first_at() + sequences + 1];
        CHECK(n == (int)seqs.size() && book.batch_size() == n);
        int row = 0;
        for (int b = 0; b < n; b++) {
            const int s = words[book.batch_at() + b], first = words[book.first_at() + b], end = words[book.first_at() + b + 1];
            CHECK(s == seqs[b] && first == row && end - first == counts[b]);
            row = end;
            for (int r = first; r < end; r++) {
                const int pos = words[s] - (end - r);
                CHECK(pos == (int)want[s].size());
                want[s].push_back(next);
                pool[(size_t)words[book.table_at() + (size_t)s * book.pitch() + pos / page_tokens] * page_tokens + pos % page_tokens] = next++;
            }
        }
        CHECK(book.batch_rows() == row);
    }
    void fork(int source, const std::vector<int>& to, int tokens) {
        book.fork(source, (int)to.size(), to.data(), tokens);
        const int n = book.list(to[0]).size();
        for (int t : to)   // (a kernel copies the rows of the lists)
            for (int i = 0; i < n; i++) words[book.table_at() + (size_t)t * book.pitch() + i] = words[book.table_at() + (size_t)source * book.pitch() + i];
        flush();
        for (int t : to) want[t].assign(want[source].begin(), want[source].begin() + (tokens < 0 ? want[source].size() : tokens));
    }
    void check() {
        CHECK(words == book.words);
        std::map<int, int> count;
        for (int s = 0; s < sequences; s++) {
            CHECK(words[s] == (int)want[s].size() && book.length(s) == words[s]);
            CHECK((int)book.list(s).size() == (words[s] + page_tokens - 1) / page_tokens);
            for (size_t i = 0; i < want[s].size(); i++) {
                const int page = words[book.table_at() + (size_t)s * book.pitch() + i / page_tokens];
                CHECK(page == book.list(s)[i / page_tokens] && page >= 0 && page < pages);
                CHECK(pool[(size_t)page * page_tokens + i % page_tokens] == want[s][i]);
            }
            for (int p : book.list(s)) count[p]++;
        }
        bool shares = false;
        for (auto& x : count) shares = shares || x.second > 1;
        CHECK(book.shares() == shares);
        CHECK(book.pages_used() == (int)count.size() && book.pages_free() == pages - (int)count.size());
    }
    template <class F>
    bool refused(F&& f, bool* full = nullptr) {
        const std::vector<int> before = words;
        try {
            f();
        } catch (const PageBook::Refused& r) {
            if (full) *full = r.full;
            CHECK(!r.why.empty() && book.changes().empty() && book.words == before);
            return true;
        }
        return false;
    }
};

static void random_run(unsigned seed) {
    std::mt19937 rng(seed);
    auto upto = [&](int n) { return (int)(rng() % (n + 1)); };
    const int page_tokens = 8 << upto(2), sequences = 2 + upto(7), pages = 4 + upto(40);
    const int most = upto(1) ? pages * page_tokens : std::max(1, pages * page_tokens / 2);
    Model m(pages, sequences, page_tokens, most);
    for (int i = 0; i < 400; i++) {
        std::vector<int> all(sequences), live, dead;
        for (int s = 0; s < sequences; s++) all[s] = s;
        std::shuffle(all.begin(), all.end(), rng);
        for (int s : all) (m.want[s].empty() ? dead : live).push_back(s);
        switch (upto(6)) {
            case 0: case 1: case 2: {
                std::vector<int> who(all.begin(), all.begin() + upto(sequences)), counts;
                for (size_t k = 0; k < who.size(); k++) counts.push_back(upto(3) ? upto(3) : upto(3 * page_tokens));
                bool full = false;
                auto want = m.want;
                if (m.refused([&] { m.extend(who, counts); }, &full)) CHECK(m.want == want);
                break;
            }
            case 3:
                if (!live.empty() && !dead.empty()) {
                    dead.resize(1 + upto((int)dead.size() - 1));
                    m.fork(live[0], dead, upto(1) ? -1 : upto((int)m.want[live[0]].size()));
                }
                break;
            case 4:
                if (!live.empty() && !dead.empty()) {
                    dead.resize(1 + upto((int)dead.size() - 1));
                    std::vector<int> from;
                    for (size_t k = 0; k < dead.size(); k++) from.push_back(live[upto((int)live.size() - 1)]);
                    if (!m.refused([&] { m.moved(m.book.copy((int)dead.size(), from.data(), dead.data())); })) {
                        m.flush();
                        for (size_t k = 0; k < dead.size(); k++) m.want[dead[k]] = m.want[from[k]];
                    }
                }
                break;
            case 5: {
                std::vector<int> who(all.begin(), all.begin() + upto(2)), keep;
                for (int s : who) keep.push_back(upto(1) ? 0 : upto((int)m.want[s].size()));
                m.book.truncate((int)who.size(), who.data(), keep.data());
                m.flush();
                for (size_t k = 0; k < who.size(); k++) m.want[who[k]].resize(keep[k]);
                break;
            }
            case 6:
                m.moved(m.book.compact());
                m.flush();
                for (int s = 0; s < sequences; s++)
                    for (int p : m.book.list(s)) CHECK(p < m.book.pages_used());
                break;
        }
        m.check();
    }
}

static void refusals() {
    Model m(4, 3, 8, 24);
    m.extend({0, 1}, {9, 8});
    m.check();
    bool full = false;
    const int out[] = {3}, low[] = {-1}, twice[] = {1, 1}, one[] = {1}, two[] = {2}, zero[] = {0}, counts[] = {1, 1}, minus[] = {-1}, far[] = {16}, near[] = {15}, many[] = {17};
    CHECK(m.refused([&] { m.book.extend(1, out, counts); }));
    CHECK(m.refused([&] { m.book.extend(1, low, counts); }));
    CHECK(m.refused([&] { m.book.extend(2, twice, counts); }));
    CHECK(m.refused([&] { m.book.extend(4, twice, counts); }));
    CHECK(m.refused([&] { m.book.extend(-1, twice, counts); }));
    CHECK(m.refused([&] { m.book.extend(1, zero, minus); }));
    CHECK(m.refused([&] { m.book.extend(1, zero, far); }, &full) && !full);    // beyond the most of one sequence
    CHECK(m.refused([&] { m.book.extend(1, two, many); }, &full) && !full ? false : full);   // more than the pages that are left
    CHECK(m.refused([&] { m.book.fork(0, 1, one, -1); }));    // has tokens
    CHECK(m.refused([&] { m.book.fork(0, 1, zero, -1); }));   // itself
    CHECK(m.refused([&] { m.book.fork(0, 1, two, 10); }));    // more tokens than there are
    CHECK(m.refused([&] { m.book.fork(3, 1, two, 0); }));
    CHECK(m.refused([&] { m.book.copy(1, zero, two); }, &full) && full);
    CHECK(m.refused([&] { m.book.copy(1, out, two); }));
    CHECK(m.refused([&] { m.book.copy(1, two, two); }));
    CHECK(m.refused([&] { m.book.copy(1, zero, one); }));
    CHECK(m.refused([&] { m.book.truncate(1, zero, near); }));
    CHECK(m.refused([&] { m.book.truncate(1, zero, minus); }));
    CHECK(m.refused([&] { m.book.truncate(2, twice, counts); }));
    m.check();
}

// Branches of one sequence that go on in one call: each but the last to have the page takes a copy of it.
static void branches() {
    Model m(8, 4, 8, 64);
    m.extend({0}, {11});
    m.fork(0, {1, 2, 3}, -1);
    m.check();
    CHECK(m.book.pages_used() == 2);
    m.extend({2, 0, 1, 3}, {1, 1, 1, 1});
    m.check();
    CHECK(m.book.pages_used() == 5);
    // as many pages as that takes, and one fewer
    Model n(5, 4, 8, 40), o(4, 4, 8, 32);
    n.extend({0}, {11});
    n.fork(0, {1, 2, 3}, -1);
    n.extend({0, 1, 2, 3}, {1, 1, 1, 1});
    n.check();
    o.extend({0}, {11});
    o.fork(0, {1, 2, 3}, -1);
    const int who[] = {0, 1, 2, 3}, counts[] = {1, 1, 1, 1};
    bool full = false;
    CHECK(o.refused([&] { o.book.extend(4, who, counts); }, &full) && full);
    o.check();
    // the batch ends with one of its sequences
    CHECK(n.book.batch_rows() == 4);
    const int two[] = {2}, three[] = {3};
    n.book.truncate(1, two, three);
    n.flush();
    CHECK(n.book.batch_size() == 0 && n.book.batch_rows() == 0);
}

// Pages that all sequences of a batch begin with, at random.
static void common(unsigned seed) {
    std::mt19937 gen(seed);
    auto upto = [&](int n) { return (int)(gen() % (unsigned)(n + 1)); };
    Model m(900, 6, 8, 1000);
    m.extend({0}, {40 + upto(60)});
    CHECK(m.book.common_pages() == 0);   // (one sequence)
    for (int s = 1; s < 5; s++) m.fork(upto(s - 1), {s}, upto(3) ? -1 : 20);
    m.extend({5}, {30});
    for (int round = 0; round < 20; round++) {
        std::vector<int> seqs = {0, 1, 2, 3, 4, 5}, counts;
        std::shuffle(seqs.begin(), seqs.end(), gen);
        seqs.resize(upto(6));
        int want = 0;
        for (int again = upto(3); again >= 0; again--) {   // (the same batch some times)
            counts.clear();
            for (size_t i = 0; i < seqs.size(); i++) counts.push_back(upto(2) ? upto(1) : upto(9));
            m.extend(seqs, counts);
            want = 0;
            while (seqs.size() > 1) {
                bool all = true;
                for (int s : seqs) all = all && want < (int)m.book.list(s).size() && m.book.list(s)[want] == m.book.list(seqs[0])[want];
                if (!all) break;
                want++;
            }
            CHECK(m.book.common_pages() == want);
            if (upto(9) == 0 && !seqs.empty()) {   // one of them is cut, or ends and becomes a branch of another
                const int s = seqs[upto((int)seqs.size() - 1)], other = (s + 1 + upto(4)) % 6, keep = upto(1) ? 0 : m.book.length(s) / 2;
                m.book.truncate(1, &s, &keep);
                m.flush();
                m.want[s].resize(keep);
                if (!keep && m.book.length(other)) m.fork(other, {s}, upto(1) ? -1 : m.book.length(other) / 2);
                m.check();
                want = m.book.common_pages();
            }
        }
        m.moved(m.book.compact());
        m.flush();
        m.check();
        CHECK(m.book.common_pages() == want);
    }
}

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "random") for (unsigned s = 0; s < 200; s++) random_run(s);
    else if (what == "refusals") refusals();
    else if (what == "branches") branches();
    else if (what == "common") for (unsigned s = 0; s < 50; s++) common(s);
    else return 2;
    return 0;
}
