// Who has which pages: the host's side of a cache of keys and values.  Lists of pages per sequence, counts of the sequences
// that share a page, and the int32 words that the kernels read (the device holds a copy of `words`).  No GPU in here.
//
// Every call checks all of its arguments first and changes nothing when it fails.
#pragma once
#include <algorithm>
#include <cstdint>
#include <exception>
#include <string>
#include <utility>
#include <vector>

namespace fynhip {

class PageBook {
  public:
    struct Refused : public std::exception {
        Refused(bool f, std::string w) : full(f), why(std::move(w)) {}
        const char* what() const noexcept override { return why.c_str(); }
        bool full;   // no pages left (else: an argument is wrong)
        std::string why;
    };
    typedef std::vector<std::pair<int, int>> Moves;   // pages to copy, from -> to: no page is both

    PageBook(int pages, int sequences, int page_tokens, int most_tokens)
        : pages_(pages), sequences_(sequences), page_tokens_(page_tokens), most_tokens_(most_tokens), pitch_((most_tokens + page_tokens - 1) / page_tokens),
          lists_(sequences), shared_(pages, 0), mark_(sequences, 0) {
        for (int i = pages - 1; i >= 0; i--) free_.push_back(i);
        words.assign((size_t)table_at() + (size_t)sequences * pitch_, 0);
    }

    // the words: tokens of each sequence | the batch's sequences | rows at which their new tokens begin, and the number of
    // sequences in the batch | lists of pages
    int batch_at() const { return sequences_; }
    int first_at() const { return 2 * sequences_; }
    size_t table_at() const { return ((size_t)3 * sequences_ + 2 + 3) / 4 * 4; }
    int pitch() const { return pitch_; }
    int length(int s) const { return words[s]; }
    int batch_size() const { return words[first_at() + sequences_ + 1]; }
    int batch_rows() const { return words[first_at() + batch_size()]; }
    int pages_free() const { return (int)free_.size(); }
    int pages_used() const { return pages_ - (int)free_.size(); }
    int common_pages() const { return common_; }                  // that all sequences of the batch begin with
    bool shares() const { return entries_ > pages_used(); }   // some page is in two lists
    int pages_of(int tokens) const { return (int)(((int64_t)tokens + page_tokens_ - 1) / page_tokens_); }
    const std::vector<int>& list(int s) const { return lists_[s]; }

    // Room for new tokens behind those of each sequence; they become the batch.  A last page that is not full and that
    // another sequence has too is copied first.
    Moves extend(int n, const int* seqs, const int* counts) {
        check(n, seqs, "extend");
        int64_t need = 0, rows = 0;
        std::vector<std::pair<int, int>> left;   // copies that this call takes off a page, while the others are counted
        for (int i = 0; i < n; i++) {
            const int s = seqs[i], len = words[s];
            if (counts[i] < 0 || counts[i] > most_tokens_ - len)
                refuse(false, "sequence " + std::to_string(s) + " has " + std::to_string(len) + " tokens, " + std::to_string(counts[i]) + " more are not within 0 and " + std::to_string(most_tokens_));
            rows += counts[i];
            need += pages_of(len + counts[i]) - pages_of(len);
            if (counts[i] > 0 && len % page_tokens_ != 0) {
                const int last = lists_[s].back();
                auto it = std::find_if(left.begin(), left.end(), [&](const std::pair<int, int>& x) { return x.first == last; });
                if (shared_[last] - (it == left.end() ? 0 : it->second) > 1) {
                    need++;
                    if (it == left.end()) left.push_back({last, 1});
                    else it->second++;
                }
            }
        }
        if (rows > 0x7fffffff) refuse(false, "too many tokens in one batch");
        if (need > (int64_t)free_.size()) refuse(true, std::to_string(need) + " pages are wanted, " + std::to_string(free_.size()) + " are free");
        // (the batch as before: of the pages in common only the last one, which need not be full, may have become a copy)
        const bool same = n > 1 && batch_size() == n && std::equal(seqs, seqs + n, words.begin() + batch_at());
        const int known = same ? std::max(0, common_ - 1) : 0;
        Moves moves;
        for (int i = 0; i < n; i++) {
            const int s = seqs[i], len = words[s];
            if (counts[i] > 0 && len % page_tokens_ != 0) {
                const int last = lists_[s].back();
                if (shared_[last] > 1) {
                    lists_[s].back() = take();
                    shared_[last]--;
                    moves.push_back({last, lists_[s].back()});
                    put(entry(s, lists_[s].size() - 1), lists_[s].back());
                }
            }
            while ((int)lists_[s].size() < pages_of(len + counts[i])) {
                lists_[s].push_back(take());
                entries_++;
                put(entry(s, lists_[s].size() - 1), lists_[s].back());
            }
        }
        for (int i = 0; i < n; i++) put(seqs[i], words[seqs[i]] + counts[i]);
        for (int i = 0; i < n; i++) put(batch_at() + i, seqs[i]);
        int row = 0;
        for (int i = 0; i < n; i++) {
            put(first_at() + i, row);
            row += counts[i];
        }
        put(first_at() + n, row);
        put(first_at() + sequences_ + 1, n);
        common_ = n > 1 ? (int)lists_[seqs[0]].size() : 0;
        for (int i = 1; i < n && common_ > 0; i++) {
            const std::vector<int>&a = lists_[seqs[0]], &b = lists_[seqs[i]];
            const int most = std::min(common_, (int)b.size());
            common_ = (int)(std::mismatch(a.begin() + known, a.begin() + most, b.begin() + known).first - a.begin());
        }
        return moves;
    }

    // The first `tokens` tokens of a sequence (-1: all) become those of empty ones too, in the same pages.  The words of
    // the lists are not noted as changed: the rows are copies of the source's, as long as the list of a branch is.
    void fork(int source, int n, const int* targets, int tokens) {
        check(1, &source, "fork");
        check(n, targets, "fork");
        const int len = words[source];
        if (tokens == -1) tokens = len;
        if (tokens < 0 || tokens > len) refuse(false, "sequence " + std::to_string(source) + " has " + std::to_string(len) + " tokens, not " + std::to_string(tokens));
        for (int i = 0; i < n; i++) {
            if (targets[i] == source) refuse(false, "a sequence cannot become a branch of itself");
            empty(targets[i]);
        }
        const int pages = pages_of(tokens);
        for (int i = 0; i < n; i++) {
            const int t = targets[i];
            lists_[t].assign(lists_[source].begin(), lists_[source].begin() + pages);
            for (int p : lists_[t]) shared_[p]++;
            entries_ += pages;
            std::copy(lists_[t].begin(), lists_[t].end(), words.begin() + entry(t, 0));
            put(t, tokens);
        }
        leave_batch(n, targets);
    }

    // Sequences become copies of others, in pages of their own.
    Moves copy(int n, const int* sources, const int* targets) {
        check(n, targets, "copy");
        int64_t need = 0;
        for (int i = 0; i < n; i++) {
            if (sources[i] < 0 || sources[i] >= sequences_) refuse(false, "copy: there is no sequence " + std::to_string(sources[i]));
            empty(targets[i]);
            need += (int64_t)lists_[sources[i]].size();
        }
        for (int i = 0; i < n; i++) mark_[targets[i]] = 1;
        bool both = false;
        for (int i = 0; i < n; i++) both = both || mark_[sources[i]];
        for (int i = 0; i < n; i++) mark_[targets[i]] = 0;
        if (both) refuse(false, "copy: a sequence is both source and target");
        if (need > (int64_t)free_.size()) refuse(true, std::to_string(need) + " pages are wanted, " + std::to_string(free_.size()) + " are free");
        Moves moves;
        for (int i = 0; i < n; i++) {
            const int t = targets[i];
            for (int p : lists_[sources[i]]) {
                lists_[t].push_back(take());
                entries_++;
                moves.push_back({p, lists_[t].back()});
                put(entry(t, lists_[t].size() - 1), lists_[t].back());
            }
            put(t, words[sources[i]]);
        }
        leave_batch(n, targets);
        return moves;
    }

    // Sequences are shortened to their first tokens; pages that none has any more are free.
    void truncate(int n, const int* seqs, const int* tokens) {
        check(n, seqs, "truncate");
        for (int i = 0; i < n; i++)
            if (tokens && (tokens[i] < 0 || tokens[i] > words[seqs[i]]))
                refuse(false, "sequence " + std::to_string(seqs[i]) + " has " + std::to_string(words[seqs[i]]) + " tokens and is not shortened to " + std::to_string(tokens[i]));
        for (int i = 0; i < n; i++) {
            const int s = seqs[i], keep = tokens ? tokens[i] : 0;
            while ((int)lists_[s].size() > pages_of(keep)) {
                const int p = lists_[s].back();
                lists_[s].pop_back();
                entries_--;
                if (--shared_[p] == 0) free_.push_back(p);
            }
            put(s, keep);
        }
        leave_batch(n, seqs);
    }

    // Used pages move into the free ones below them until they are the first ones of all.
    Moves compact() {
        const int used = pages_used();
        Moves moves;
        std::vector<int> to(pages_, -1);
        int hole = 0;
        for (int p = pages_ - 1; p >= used; p--) {
            if (!shared_[p]) continue;
            while (shared_[hole]) hole++;
            to[p] = hole;
            shared_[hole] = shared_[p];
            shared_[p] = 0;
            moves.push_back({p, hole});
        }
        if (!moves.empty())
            for (int s = 0; s < sequences_; s++)
                for (size_t i = 0; i < lists_[s].size(); i++)
                    if (to[lists_[s][i]] >= 0) {
                        lists_[s][i] = to[lists_[s][i]];
                        put(entry(s, i), lists_[s][i]);
                    }
        free_.clear();
        for (int p = pages_ - 1; p >= used; p--) free_.push_back(p);
        return moves;
    }

    // Sequences whose tokens a caller wants to have: that there are such.
    void check(int n, const int* seqs, const char* what) {
        if (n < 0 || n > sequences_) refuse(false, std::string(what) + ": " + std::to_string(n) + " sequences, the cache has " + std::to_string(sequences_));
        if (n > 0 && !seqs) refuse(false, std::string(what) + ": no sequences given");
        int i = 0;
        for (; i < n; i++) {
            if (seqs[i] < 0 || seqs[i] >= sequences_ || mark_[seqs[i]]) break;
            mark_[seqs[i]] = 1;
        }
        for (int k = 0; k < i; k++) mark_[seqs[k]] = 0;
        if (i == n) return;
        if (seqs[i] < 0 || seqs[i] >= sequences_) refuse(false, std::string(what) + ": there is no sequence " + std::to_string(seqs[i]));
        refuse(false, std::string(what) + ": sequence " + std::to_string(seqs[i]) + " is named twice");
    }

    std::vector<int32_t> words;
    // changes of the words since the last call of changes_taken(), as [first, behind the last) in the order they were made
    const std::vector<std::pair<size_t, size_t>>& changes() const { return changes_; }
    void changes_taken() { changes_.clear(); }

  private:
    int pages_, sequences_, page_tokens_, most_tokens_, pitch_;
    int64_t entries_ = 0;       // of all lists
    int common_ = 0;
    std::vector<std::vector<int>> lists_;
    std::vector<int> shared_;   // sequences that have a page
    std::vector<int> free_;     // (a stack: the page that was freed last is taken first)
    std::vector<char> mark_;
    std::vector<std::pair<size_t, size_t>> changes_;

    [[noreturn]] static void refuse(bool full, const std::string& why) { throw Refused(full, why); }
    void empty(int s) {
        if (words[s] != 0) refuse(false, "sequence " + std::to_string(s) + " has tokens already");
    }
    int take() {
        const int p = free_.back();
        free_.pop_back();
        shared_[p] = 1;
        return p;
    }
    size_t entry(int s, size_t i) const { return table_at() + (size_t)s * pitch_ + i; }
    void put(size_t at, int v) {
        if (words[at] == v) return;
        words[at] = v;
        if (!changes_.empty() && changes_.back().second == at) changes_.back().second++;
        else changes_.push_back({at, at + 1});
    }
    // The tokens of the batch are at the ends of its sequences: where one is cut, replaced or emptied there is no batch.
    void leave_batch(int n, const int* seqs) {
        const int have = batch_size();
        if (!have || !n) return;
        for (int i = 0; i < n; i++) mark_[seqs[i]] = 1;
        bool hit = false;
        for (int i = 0; i < have; i++) hit = hit || mark_[words[batch_at() + i]];
        for (int i = 0; i < n; i++) mark_[seqs[i]] = 0;
        if (!hit) return;
        put(first_at(), 0);
        put(first_at() + sequences_ + 1, 0);
    }
};

}  // namespace fynhip
